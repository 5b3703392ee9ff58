// C (M, N) = A (M, K) . B (N, K)^T + bias with both operands packed MXFP4
// (mxfp4.h), on the block-scaled 16x16x128 MFMA with fp32 accumulators.
//
// Bounds, measured (MI355X, packed operands, weights from HBM):
//   one row of the largest tile on every CU and more: the matrix cores at the clock that the power allows. The
//   instruction alone sustains 6.4 to 7.1 PFLOP/s; (16384, 5120, 13824) runs at 4.7 (5.1 at best), (32768, 13824, 5120)
//   at 4.2 to 4.5, of which the stores of a tile, 128 KB a CU that no other tile's work covers, take 11%.
//   up to some hundred rows: the operands' way from HBM through one workgroup's ring, 50 to 60 GB/s a CU, in one
//   round of workgroups: (154, 10240, 4096) 11.2 us with 22 MB of weights, (1024, 5120, 5120) 21.5 us.
#include <algorithm>
#include <type_traits>

#include "featherops_amd.h"
#include "lds_dma.h"
#include "mxfp4.h"

namespace feather {
namespace {

// dma16_lds, and the same for 4 bytes per lane, with an offset that the instruction adds to both addresses:
// copies a KB apart in LDS share one M0.
template <int kOffset>
__device__ __forceinline__ void dma16_lds_at(const void* sbase, uint32_t voff, uint32_t lds_addr) {
    static_assert(kOffset >= 0 && kOffset < 4096, "instruction offset");
    asm volatile(
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %1 offset:%3"
        :
        : "v"(voff), "s"(sbase), "{m0}"(lds_addr), "n"(kOffset)
        : "memory");
}
__device__ __forceinline__ void dma4_lds(const void* sbase, uint32_t voff, uint32_t lds_addr) {
    asm volatile(
        "s_nop 0\n\t"
        "global_load_lds_dword %0, %1"
        :
        : "v"(voff), "s"(sbase), "{m0}"(lds_addr)
        : "memory");
}

// A wave-uniform pointer in scalar registers, as the copies take it.
__device__ __forceinline__ const uint8_t* scalar_pointer(const uint8_t* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v)));
    const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32)));
    return reinterpret_cast<const uint8_t*>(hi << 32 | lo);
}

struct TileArgs {
    const uint8_t* a;
    const uint8_t* as;
    const uint8_t* b;
    const uint8_t* bs;
    const uint16_t* bias;
    uint16_t* c;
    int64_t M, ldc;  // rows of this launch, elements between rows of c
    int N, ksteps, a_groups, b_groups;
    int tiles_m, tiles_n, ksplit, group_m;
    uint32_t* counters;
    float* partials;
};

// One workgroup computes a BM x BN tile of C over its share of the K steps with
// WM x WN waves. The weights take the MFMA's first operand, so a lane ends with
// four consecutive columns of one row of C and stores them together.
//
// Per K step the tile's operands (BM + BN rows of 64 bytes, and a dword of scales
// per lane and 64 rows) are copied from HBM into a ring of kStages LDS buffers; a
// fragment is one contiguous KB in HBM, in LDS and in the wave's ds_read_b128, so
// there is no swizzle and no bank conflict. Every iteration waits for the stage
// after the one it multiplies, issues the copies of the stage kStages - 1 ahead into the
// buffer it has emptied, and reads the next stage's fragments into the other half
// of its fragment registers under this stage's MFMAs. Copies past the last step
// repeat it, so the wait counts are constants.
template <int BM, int BN, int WM, int WN, int kStages, bool kBf16>
__global__ __launch_bounds__(64 * WM * WN, 2) void mx_tile_kernel(const TileArgs p) {
    constexpr int kWaves = WM * WN;
    constexpr int TM = BM / WM, TN = BN / WN;  // wave tile
    constexpr int FM = TM / 16, FN = TN / 16;  // its fragments
    constexpr int kGroupsM = BM / 64, kGroupsN = BN / 64;
    constexpr int kCodeCopies = (BM + BN) / 16, kScaleCopies = kGroupsM + kGroupsN;
    constexpr int kCodes = kCodeCopies / kWaves, kScales = (kScaleCopies + kWaves - 1) / kWaves;
    constexpr int kPerWave = kCodes + kScales;  // copies of a stage by every wave (surplus scales repeat the last)
    constexpr int kStageBytes = kCodeCopies * 1024 + kScaleCopies * 256;
    constexpr int kScaleBase = kCodeCopies * 1024;
    constexpr int SM = (FM + 3) / 4, SN = (FN + 3) / 4;  // scale dwords of the wave's rows and columns
    static_assert(kStages * kStageBytes <= 160 * 1024 && kStages % 2 == 0, "LDS");
    static_assert(kCodeCopies % kWaves == 0 && kCodes <= 4, "copies");
    static_assert((kStages - 1) * kPerWave < 64, "vmcnt range");
    static_assert(FM % 2 == 0 && FN % 2 == 0 && (FM % 4 == 0 || FM == 2) && (FN % 4 == 0 || FN == 2), "scale bytes");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kStages * kStageBytes];

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int wm = wave / WN, wn = wave % WN;

    // Workgroup -> tile: an XCD's workgroups (p % 8) take a contiguous run of the raster, which walks
    // group_m tile rows at a time, so an XCD's L2 holds few rows and columns of tiles at once.
    const int total = p.tiles_m * p.tiles_n * p.ksplit;
    const int xcd = blockIdx.x % kNumXcd;
    const int run = total / kNumXcd, more = total % kNumXcd;
    const int t = xcd * run + min(xcd, more) + blockIdx.x / kNumXcd;
    const int q = t % p.ksplit;
    const int lin = t / p.ksplit;
    const int per_group = p.group_m * p.tiles_n;
    const int first_m = lin / per_group * p.group_m;
    const int rows_here = min(p.group_m, p.tiles_m - first_m);
    const int tm = first_m + lin % per_group % rows_here;
    const int tn = lin % per_group / rows_here;
    const int64_t m0 = static_cast<int64_t>(tm) * BM;
    const int n0 = tn * BN;
    const int k0 = static_cast<int>(static_cast<int64_t>(p.ksteps) * q / p.ksplit);
    const int steps = static_cast<int>(static_cast<int64_t>(p.ksteps) * (q + 1) / p.ksplit) - k0;

    // This wave's copies: their addresses at step k0. Groups of 64 rows past an operand's end read its last one.
    const uint8_t* src[kPerWave];
    const uint32_t lds = lds_addr_of(smem);
    const uint32_t code_dst = lds + wave * (kCodes * 1024);
    uint32_t scale_dst[kScales];
#pragma unroll
    for (int i = 0; i < kCodes; ++i) {
        const int j = wave * kCodes + i;
        const bool is_a = j < BM / 16;
        const int f = is_a ? j : j - BM / 16;
        const int64_t g = is_a ? min(static_cast<int>(m0 / 64) + f / 4, p.a_groups - 1) : min(n0 / 64 + f / 4, p.b_groups - 1);
        src[i] = scalar_pointer((is_a ? p.a : p.b) + ((g * p.ksteps + k0) * 4 + f % 4) * 1024 - i * 1024);  // (see copy)
    }
#pragma unroll
    for (int i = 0; i < kScales; ++i) {
        const int j = min(i * kWaves + wave, kScaleCopies - 1);
        const bool is_a = j < kGroupsM;
        const int64_t g = is_a ? min(static_cast<int>(m0 / 64) + j, p.a_groups - 1) : min(n0 / 64 + j - kGroupsM, p.b_groups - 1);
        src[kCodes + i] = scalar_pointer((is_a ? p.as : p.bs) + (g * p.ksteps + k0) * 256);
        scale_dst[i] = lds + kScaleBase + j * 256;
    }
    // (the step in the lane's offset, one instruction for all copies, not in each copy's address)
    auto copy = [&](auto i, int step, int slot) {
        if constexpr (i < kCodes) dma16_lds_at<i * 1024>(src[i], lane * 16 + step * 4096, code_dst + slot * kStageBytes);
        else dma4_lds(src[i], lane * 4 + step * 256, scale_dst[i - kCodes] + slot * kStageBytes);
    };

    struct Frags {
        uint4 a[FM], b[FN];
        uint32_t sa[SM], sb[SN];
    };
    constexpr int kReads = SM + SN + FM + FN;
    auto read = [&](auto r, Frags& f, const uint8_t* base) {
        if constexpr (r < SN) {
            f.sb[r] = *reinterpret_cast<const uint32_t*>(base + kScaleBase + (kGroupsM + wn * TN / 64 + r) * 256 + lane * 4);
        } else if constexpr (r < SN + SM) {
            constexpr int i = r - SN;
            f.sa[i] = *reinterpret_cast<const uint32_t*>(base + kScaleBase + (wm * TM / 64 + i) * 256 + lane * 4);
        } else if constexpr (r < SN + SM + FN) {
            constexpr int i = r - SN - SM;
            f.b[i] = *reinterpret_cast<const uint4*>(base + (BM / 16 + wn * FN + i) * 1024 + lane * 16);
        } else {
            constexpr int i = r - SN - SM - FN;
            f.a[i] = *reinterpret_cast<const uint4*>(base + (wm * FM + i) * 1024 + lane * 16);
        }
    };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // (half a group's scales are moved down where they are used: beside the read they would wait for it)
    auto multiply = [&](auto n, const Frags& f) {
        constexpr int i = n / FN, j = n % FN;
        const uint32_t sb = FN == 2 ? f.sb[0] >> (16 * (wn % 2)) : f.sb[j / 4];
        const uint32_t sa = FM == 2 ? f.sa[0] >> (16 * (wm % 2)) : f.sa[i / 4];
        acc[i][j] = mfma_mx<j % 4, i % 4>(f.b[j], f.a[i], acc[i][j], sb, sa);
    };

#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) unrolled<kPerWave>([&](auto i) { copy(i, min(s, steps - 1), s); });
    Frags f0, f1;
    wait_vmcnt<(kStages - 2) * kPerWave>();
    stage_barrier();
    unrolled<kReads>([&](auto r) { read(r, f0, smem); });
    // One step, in ring buffer `slot`. The loop below goes round the ring, so that buffers' addresses are
    // constants (256 x 256: 70.9 -> 68.5 us at M 4096, N = K = 5120; the small tiles the same).
    // The copies and the next step's reads are pinned between the MFMAs, all of them in the
    // first three quarters: left alone, the compiler reads each fragment into the registers of the one
    // just used up, after its last MFMA, and every step waits for LDS with the matrix cores idle.
    constexpr int kMfmas = FM * FN, kOps = kPerWave + kReads, kOver = kMfmas >= 8 ? kMfmas * 3 / 4 : kMfmas;
    auto iterate = [&](auto slot, int k, const Frags& now, Frags& next) {
        constexpr int kAfter = (slot + 1) % kStages, kFree = (slot + kStages - 1) % kStages;
        const int ahead = min(k + kStages - 1, steps - 1);
        const uint8_t* base = smem + kAfter * kStageBytes;
        // Stage k + 1 has landed; the buffer of stage k - 1 is free: the MFMAs of that step, which are
        // issued, waited for its reads. The reads of stage k may still be under way.
        wait_vmcnt<(kStages - 3) * kPerWave>();
        stage_barrier();
        unrolled<kMfmas>([&](auto n) {
            multiply(n, now);
            constexpr int first = n < kOver ? n * kOps / kOver : kOps, last = n < kOver ? (n + 1) * kOps / kOver : kOps;
            unrolled<last - first>([&](auto o) {
                // the copies in even steps among the reads
                constexpr int op = first + o, copies = (op + 1) * kPerWave / kOps, before = op * kPerWave / kOps;
                if constexpr (copies > before) copy(std::integral_constant<int, before>{}, ahead, kFree);
                else read(std::integral_constant<int, op - before>{}, next, base);
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    for (int k = 0; k < steps; k += kStages) {
        unrolled<kStages>([&](auto slot) {
            if (k + slot >= steps) return;
            if constexpr (slot % 2 == 0) iterate(slot, k + slot, f0, f1);
            else iterate(slot, k + slot, f1, f0);
        });
    }
    wait_vmcnt<0>();

    const int lm = lane & 15;
    if (p.ksplit > 1) {
        // Each split writes its fp32 accumulators to the workspace in fragment order and counts itself
        // in; the last to arrive adds the splits' sums in split order and goes on to the epilogue.
        // Ordering: the partials are written and read with agent-scope (sc1) accesses alone, which
        // are coherent across the XCDs. A store is acknowledged (vmcnt) once it is visible at agent
        // scope; every wave waits for that before the barrier that precedes the arrival count, and
        // the last arrival's loads depend on the count's answer.
        constexpr int kTileBytes = BM * BN * 4;
        constexpr int kCoherent = 16;  // sc1
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        const __amdgpu_buffer_rsrc_t prs = __builtin_amdgcn_make_buffer_rsrc(
            p.partials + static_cast<int64_t>(lin) * p.ksplit * (kTileBytes / 4), 0, p.ksplit * kTileBytes, 0x00020000);
        auto at = [&](int i, int j) { return (((wave * FM + i) * FN + j) * 64 + lane) * 16; };
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[i][j]), prs, q * kTileBytes + at(i, j), 0, kCoherent);
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        __shared__ int last_flag;
        __syncthreads();
        if (tid == 0)
            last_flag = __hip_atomic_fetch_add(&p.counters[lin], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                        static_cast<uint32_t>(p.ksplit - 1);
        __syncthreads();
        if (!last_flag) return;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < p.ksplit; ++s) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] += __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(prs, s * kTileBytes + at(i, j), 0, kCoherent));
        }
        if (tid == 0)  // ready for the next call on this stream
            __hip_atomic_store(&p.counters[lin], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }

    // Epilogue: bias added in fp32, one rounding to the output type. A lane has four columns of each
    // fragment; neighbouring quarters of the wave (lane ^ 16) trade one fragment of a pair for the other,
    // so that every lane stores 8 columns and a row gets 64 contiguous bytes from one instruction. (Rows of C off
    // 16-byte boundaries, N no multiple of 8, make unaligned stores: 3844 x 7679 x 722 45 us, x 7676 28, x 7680 25.)
    const int kb = lane >> 4;
    unrolled<FN / 2>([&](auto h) {
        constexpr int j = 2 * h;
        const int n = n0 + wn * TN + (j + (kb & 1)) * 16 + (kb >> 1) * 8;  // after the trade
        float bias[2][4] = {};
        if (p.bias) {
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    bias[f][e] = out_bits_to_f32<kBf16>(p.bias[min(n0 + wn * TN + (j + f) * 16 + kb * 4 + e, p.N - 1)]);
        }
        unrolled<FM>([&](auto i) {
            const int64_t m = m0 + wm * TM + i * 16 + lm;
            uint32_t o[2][2];
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    o[f][e] = mx_round_pair<kBf16>(acc[i][j + f][2 * e] + bias[f][2 * e], acc[i][j + f][2 * e + 1] + bias[f][2 * e + 1]);
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const auto r = __builtin_amdgcn_permlane16_swap(o[0][e], o[1][e], false, false);
                v[e] = r[0];
                v[2 + e] = r[1];
            }
            if (m >= p.M || n >= p.N) return;
            uint16_t* c = p.c + m * p.ldc + n;
            if (n + 8 <= p.N) {
                __builtin_memcpy(c, v, 16);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n + e < p.N) c[e] = static_cast<uint16_t>(v[e >> 1] >> (16 * (e & 1)));
            }
        });
    });
}

struct Tile {
    int bm, bn;
    int per_cu;   // workgroups a CU holds
    double base;  // us of a launch with next to no K
    double lo, one, two, three;  // us per K step: few workgroups, one, two, three on every CU
};
// Tiles of the plan (ids 1..) and their times, MI355X, packed operands. The constants are those with which the
// pick came nearest to the fastest of all tiles and splits, over 330 shapes (M 33 .. 6000, N 256 .. 16384, K 256 ..
// 16384), each with the weight in HBM and in the caches: 1.4% and 1.3% above it in the geometric mean, 21% and 18% at
// most. Small tiles fill the chip where there are few rows; large ones read each operand fewer times.
constexpr Tile kTiles[] = {
    {0, 0, 0, 0, 0, 0, 0, 0},
    {64, 64, 3, 4.1, 0.12, 0.16, 0.35, 0.42},
    {64, 128, 2, 4.2, 0.176, 0.23, 0.37, 0},
    {128, 128, 2, 4.1, 0.316, 0.36, 0.57, 0},
    {128, 256, 1, 5.4, 0.38, 0.54, 0, 0},
    {256, 256, 1, 6.4, 0.49, 0.93, 0, 0},
};
constexpr int kNumTiles = 6, kLargest = 5;
constexpr int kCus = 256;
// Tile rows the raster walks at a time: an XCD's 32 workgroups of the largest tile then cover about as many rows
// as columns. 4, 6, 8 at (32768, 13824, 5120): 1095, 1050, 1113 us; (2048, 5120, 5120) in 64 x 128 tiles: 46.7,
// 43.0, 44.9; M = 1024 the same within 2%.
constexpr int kRasterRows = 6;

int64_t tiles_of(int64_t n, int t) { return (n + t - 1) / t; }

// Time of `wgs` workgroups of a tile, `steps` K steps each.
double tile_time(const Tile& t, int64_t wgs, double steps) {
    const int64_t slots = static_cast<int64_t>(kCus) * t.per_cu;
    const double full = t.per_cu == 3 ? t.three : t.per_cu == 2 ? t.two : t.one;
    double time = static_cast<double>(wgs / slots) * full * steps;
    const int64_t rest = wgs % slots;
    if (rest > 2 * kCus) time += t.three * steps;
    else if (rest > kCus) time += t.two * steps;
    else if (rest > 0) time += (t.lo + (t.one - t.lo) * static_cast<double>(rest) / kCus) * steps;
    return t.base + time;
}

// The fastest tile and K split for (M, N) on its own.
struct Choice {
    int tile, ksplit;
    double time;
};
Choice choose(int64_t M, int64_t N, int64_t ksteps) {
    Choice best{1, 1, 1e30};
    for (int id = 1; id < kNumTiles; ++id) {
        const Tile& t = kTiles[id];
        const int64_t tiles = tiles_of(M, t.bm) * tiles_of(N, t.bn);
        for (int ks : {1, 2, 3, 4, 6, 8}) {
            // a split leaves every part eight steps or more, and keeps to one round of workgroups (and the
            // arrival counters' 64 KB); it costs the exchange of the partial sums
            if (ks > 1 && (ksteps / ks < 8 || tiles * ks > kCus * t.per_cu)) break;
            double time = tile_time(t, tiles * ks, static_cast<double>((ksteps + ks - 1) / ks));
            if (ks > 1) time += 1.2 + static_cast<double>(tiles * ks) * t.bm * t.bn * 8 / 4.6e6;
            if (time < best.time) best = {id, ks, time};
        }
    }
    return best;
}

size_t split_bytes(int64_t M, int64_t N, const Choice& c) {
    if (c.ksplit == 1) return 0;
    const Tile& t = kTiles[c.tile];
    return kMxCounterBytes + static_cast<size_t>(tiles_of(M, t.bm) * tiles_of(N, t.bn)) * c.ksplit * t.bm * t.bn * 4;
}

// The plan: one tile for the whole result, or whole rounds of the largest tile for its first columns (or
// rows) and the tile that suits the rest, where those would leave most of the chip idle in a last round.
struct Plan {
    int64_t m1, n1;  // the second part starts at row m1 or column n1 (the other is 0); both 0: one part
    Choice first, rest;
};
Plan make_plan(int64_t M, int64_t N, int64_t ksteps) {
    Plan best{0, 0, choose(M, N, ksteps), {}};
    const Tile& t = kTiles[kLargest];
    const int64_t tm = tiles_of(M, t.bm), tn = tiles_of(N, t.bn);
    const int64_t whole = tm * tn / kCus * kCus;
    if (whole == 0 || whole == tm * tn) return best;
    double time = best.first.time;
    for (int by_rows = 0; by_rows < 2; ++by_rows) {
        const int64_t lines = by_rows ? whole / tn : whole / tm;
        if (lines == 0) continue;
        const int64_t m1 = by_rows ? lines * t.bm : 0, n1 = by_rows ? 0 : lines * t.bn;
        if (m1 >= M || n1 >= N) continue;
        const Choice first{kLargest, 1, tile_time(t, lines * (by_rows ? tn : tm), static_cast<double>(ksteps))};
        const Choice rest = choose(M - m1, N - n1, ksteps);
        if (first.time + rest.time < time) {
            time = first.time + rest.time;
            best = {m1, n1, first, rest};
        }
    }
    return best;
}

template <int BM, int BN, int WM, int WN, int kStages>
void launch(const TileArgs& a, bool bf16, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(a.tiles_m * a.tiles_n * a.ksplit);
    if (bf16) mx_tile_kernel<BM, BN, WM, WN, kStages, true><<<grid, 64 * WM * WN, 0, stream>>>(a);
    else mx_tile_kernel<BM, BN, WM, WN, kStages, false><<<grid, 64 * WM * WN, 0, stream>>>(a);
}

// Rows [m0, M) and columns [n0, N) of the product.
int run(const MxMmArgs& p, Choice c, int64_t m0, int64_t n0, int64_t M, int64_t N, hipStream_t stream) {
    const Tile& t = kTiles[c.tile];
    if (split_bytes(M - m0, N - n0, c) > p.ws_bytes) c.ksplit = 1;
    const int64_t tiles_m = tiles_of(M - m0, t.bm), tiles_n = tiles_of(N - n0, t.bn), ksteps = mx_ksteps(p.K);
    if (tiles_m * tiles_n > (int64_t(1) << 22)) return FEATHER_ERR_UNSUPPORTED;
    const int64_t a_skip = m0 / 64 * ksteps, b_skip = n0 / 64 * ksteps;
    const TileArgs a{p.a + a_skip * 4096, p.a_scales + a_skip * 256, p.b + b_skip * 4096, p.b_scales + b_skip * 256,
                     p.bias ? p.bias + n0 : nullptr, p.c + m0 * p.N + n0, M - m0, p.N, static_cast<int>(N - n0),
                     static_cast<int>(ksteps), static_cast<int>(mx_groups(p.M) - m0 / 64),
                     static_cast<int>(mx_groups(p.N) - n0 / 64), static_cast<int>(tiles_m), static_cast<int>(tiles_n),
                     c.ksplit, kRasterRows, reinterpret_cast<uint32_t*>(p.ws), reinterpret_cast<float*>(p.ws + kMxCounterBytes)};
    switch (c.tile) {
        case 1: launch<64, 64, 2, 2, 6>(a, p.out_bf16, stream); break;
        case 2: launch<64, 128, 2, 2, 6>(a, p.out_bf16, stream); break;
        case 3: launch<128, 128, 2, 2, 4>(a, p.out_bf16, stream); break;
        case 4: launch<128, 256, 2, 4, 6>(a, p.out_bf16, stream); break;
        default: launch<256, 256, 4, 2, 4>(a, p.out_bf16, stream); break;
    }
    return hipGetLastError() == hipSuccess ? FEATHER_OK : FEATHER_ERR_LAUNCH;
}

}  // namespace

size_t mx_tiles_workspace(int64_t M, int64_t N, int64_t K) {
    const Plan plan = make_plan(M, N, mx_ksteps(K));
    if (!plan.m1 && !plan.n1) return split_bytes(M, N, plan.first);
    return split_bytes(M - plan.m1, N - plan.n1, plan.rest);
}

void mx_tiles_parts(int64_t M, int64_t N, int64_t K, int64_t* plan) {
    const Plan p = make_plan(M, N, mx_ksteps(K));
    auto part = [](int64_t* out, const Choice& c) { out[0] = kTiles[c.tile].bm, out[1] = kTiles[c.tile].bn, out[2] = c.ksplit; };
    part(plan, p.first);
    if (p.m1 || p.n1) part(plan + 3, p.rest);
    plan[6] = p.m1;
    plan[7] = p.n1;
}

int mx_mm_tiles(const MxMmArgs& p, hipStream_t stream) {
    const Plan plan = make_plan(p.M, p.N, mx_ksteps(p.K));
    if (!plan.m1 && !plan.n1) return run(p, plan.first, 0, 0, p.M, p.N, stream);
    const int st = run(p, plan.first, 0, 0, plan.m1 ? plan.m1 : p.M, plan.n1 ? plan.n1 : p.N, stream);
    return st == FEATHER_OK ? run(p, plan.rest, plan.m1, plan.n1, p.M, p.N, stream) : st;
}

}  // namespace feather
