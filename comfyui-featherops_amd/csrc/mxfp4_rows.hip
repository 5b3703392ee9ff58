// The MXFP4 product for few rows: C (M, N) = q(A) . B^T + bias, where the call is
// bound by streaming the weight once. 16-bit activations are quantised on the way
// into the matrix instruction (MxPieces: ~85 instructions a K step, beside the 1 to 4 KB of
// weights that the wave waits for); a launch of its own for the quantisation would cost
// more than that of one token's product. One row and N = 13824, K = 5120 (37.6 MB) takes 8.7 us
// on the GPU, 4.3 TB/s with the launch; 16 rows and N = K = 4096 (8.9 MB) 6.0 us, of which some
// 3 are the launch, the first load's way and the join of the eight waves.
#include <algorithm>
#include <type_traits>

#include "featherops_amd.h"
#include "mxfp4.h"

namespace feather {
namespace {

constexpr int kWaves = 8;

struct RowsArgs {
    const uint8_t* a;
    const uint8_t* as;
    int a_row_bytes;
    const uint8_t* b;
    const uint8_t* bs;
    const uint16_t* bias;
    uint16_t* c;
    int M, N, K, ksteps;
    int strips, ksplit;
    uint32_t* counters;
    float* partials;
};

// One step's operands of a wave: A fragments (packed, or as 16-bit values) and B fragments.
template <int MT, int NT, int AT>
struct Step {
    std::conditional_t<AT == kMxPacked, uint4, MxPieces<AT == kMxBf16 ? kMxBf16 : kMxF16>> a[MT];
    uint32_t as, bs;
    uint4 b[NT];
};

// A workgroup takes NT column tiles (a strip) and all MT row tiles; its waves take
// the K steps in turn, kDepth steps' loads in flight each, and add their sums
// through LDS in wave order. ksplit > 1: several workgroups share a strip's steps.
template <int MT, int NT, int AT, bool kBf16>
__global__ __launch_bounds__(64 * kWaves) void mx_rows_kernel(const RowsArgs p) {
    constexpr int kDepth = 2;
    __shared__ __attribute__((aligned(16))) f32x4 red[kWaves][MT * NT][64];
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;

    // an XCD's workgroups take neighbouring strips: up to four share their scales' cache lines
    const int total = p.strips * p.ksplit;
    const int xcd = blockIdx.x % kNumXcd;
    const int run = total / kNumXcd, more = total % kNumXcd;
    const int t = xcd * run + min(xcd, more) + blockIdx.x / kNumXcd;
    const int q = t % p.ksplit;
    const int strip = t / p.ksplit;
    const int n0 = strip * NT * 16;
    const int k0 = static_cast<int>(static_cast<int64_t>(p.ksteps) * q / p.ksplit);
    const int k1 = static_cast<int>(static_cast<int64_t>(p.ksteps) * (q + 1) / p.ksplit);

    const int64_t tile0 = static_cast<int64_t>(strip) * NT;
    const int bshift = 8 * static_cast<int>(tile0 % 4);
    typedef Step<MT, NT, AT> S;
    // Operands come through buffer descriptors: a step past the wave's last one reads nothing, so the loop
    // has no branch around loads, where the compiler would wait for all of those in flight.
    const __amdgpu_buffer_rsrc_t bres = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(p.b + (tile0 / 4 * p.ksteps * 4 + tile0 % 4) * 1024), 0,
        (p.ksteps * 4 - static_cast<int>(tile0 % 4)) * 1024, 0x00020000);
    const __amdgpu_buffer_rsrc_t bsres = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(p.bs + (tile0 / 4) * p.ksteps * 256), 0, p.ksteps * 256, 0x00020000);
    const __amdgpu_buffer_rsrc_t ares = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(p.a), 0, AT == kMxPacked ? p.ksteps * 4096 : (p.M - 1) * p.a_row_bytes + p.K * 2, 0x00020000);
    const __amdgpu_buffer_rsrc_t asres = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(AT == kMxPacked ? p.as : p.a), 0, AT == kMxPacked ? p.ksteps * 256 : 0, 0x00020000);
    constexpr uint32_t kNone = 0x80000000u;  // an offset past every descriptor's end
    uint32_t arow[MT][AT == kMxPacked ? 1 : 4];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        if constexpr (AT == kMxPacked) {
            arow[i][0] = i * 1024 + lane * 16;
        } else {  // rows past the last repeat it (their results are not stored)
#pragma unroll
            for (int v = 0; v < 4; ++v)
                arow[i][v] = min(i * 16 + mx_piece_row(lane, v), p.M - 1) * p.a_row_bytes + mx_piece_col(lane) * 2;
        }
    }
    auto load_b = [&](S& s, int k, bool have) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
            s.b[j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
                                                   bres, have ? (k * 4 + j) * 1024 + lane * 16 : kNone, 0, 0));
        s.bs = __builtin_amdgcn_raw_buffer_load_b32(bsres, have ? k * 256 + lane * 4 : kNone, 0, 0);
    };
    // a step that ends within K
    auto load = [&](S& s, int k, bool have) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if constexpr (AT == kMxPacked) {
                s.a[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(ares, have ? arow[i][0] + k * 4096 : kNone, 0, 0));
            } else {
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    s.a[i].v[v][0] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
                                                                   ares, have ? arow[i][v] + k * (kMxStepK * 2) : kNone, 0, 0));
            }
        }
        if constexpr (AT == kMxPacked) s.as = __builtin_amdgcn_raw_buffer_load_b32(asres, have ? k * 256 + lane * 4 : kNone, 0, 0);
        load_b(s, k, have);
        // the loads start here, not where the compiler would move them: beside their use, a step later
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const S& s) {
        const uint32_t bscale = NT == 4 ? s.bs : s.bs >> bshift;
        unrolled<MT>([&](auto i) {
            uint4 a;
            uint32_t ascale;
            constexpr int kByte = AT == kMxPacked ? i : 0;
            if constexpr (AT == kMxPacked) {
                a = s.a[i];
                ascale = s.as;
            } else {
                a = s.a[i].quantize(lane, &ascale);
            }
            unrolled<NT>([&](auto j) { acc[i][j] = mfma_mx<j, kByte>(s.b[j], a, acc[i][j], bscale, ascale); });
        });
    };

    const int whole = AT == kMxPacked ? k1 : min(k1, p.K / kMxStepK);  // steps before this one end within K
    const int first = k0 + wave;
    if (first < whole) {
        S buf[kDepth];
#pragma unroll
        for (int d = 0; d < kDepth; ++d) load(buf[d], first + d * kWaves, first + d * kWaves < whole);
        for (int k = first; k < whole; k += kDepth * kWaves) {
#pragma unroll
            for (int d = 0; d < kDepth; ++d) {
                if (k + d * kWaves < whole) multiply(buf[d]);
                const int next = k + (kDepth + d) * kWaves;
                load(buf[d], next, next < whole);
            }
        }
    }
    if constexpr (AT != kMxPacked) {
        if (whole < k1 && (whole - k0) % kWaves == wave) {
            S tail;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const int col = whole * kMxStepK + mx_piece_col(lane);
                    const uint8_t* row = p.a + arow[i][v] - mx_piece_col(lane) * 2;
                    if (p.K >= 8) tail.a[i].load_end(v, row, col, p.K);
                    else tail.a[i].load_few(v, row + col * 2, p.K - col);
                }
            load_b(tail, whole, true);
            multiply(tail);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) red[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();

    // Entry e of the strip's result: 4 consecutive columns of one row.
    constexpr int kEntries = MT * NT * 64;
    constexpr int kTileBytes = kEntries * 16;
    constexpr int kCoherent = 16;  // sc1
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    if (p.ksplit > 1) {
        // Partials travel as in the tile kernel: agent-scope stores, acknowledged before the count.
        const __amdgpu_buffer_rsrc_t prs = __builtin_amdgcn_make_buffer_rsrc(
            p.partials + static_cast<int64_t>(strip) * p.ksplit * (kTileBytes / 4), 0, p.ksplit * kTileBytes, 0x00020000);
        for (int e = tid; e < kEntries; e += 64 * kWaves) {
            f32x4 sum = red[0][e >> 6][e & 63];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) sum += red[w][e >> 6][e & 63];
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum), prs, q * kTileBytes + e * 16, 0, kCoherent);
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        __shared__ int last_flag;
        __syncthreads();
        if (tid == 0)
            last_flag = __hip_atomic_fetch_add(&p.counters[strip], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                        static_cast<uint32_t>(p.ksplit - 1);
        __syncthreads();
        if (!last_flag) return;
        for (int e = tid; e < kEntries; e += 64 * kWaves) {
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
            for (int s = 0; s < p.ksplit; ++s)
                sum += __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(prs, s * kTileBytes + e * 16, 0, kCoherent));
            red[0][e >> 6][e & 63] = sum;  // (read back below by this thread alone)
        }
        if (tid == 0)  // ready for the next call on this stream
            __hip_atomic_store(&p.counters[strip], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    for (int e = tid; e < kEntries; e += 64 * kWaves) {
        const int l = e & 63;
        const int m = (e >> 6) / NT * 16 + (l & 15);
        const int n = n0 + (e >> 6) % NT * 16 + (l >> 4) * 4;
        if (m >= p.M || n >= p.N) continue;
        f32x4 sum = red[0][e >> 6][l];
        if (p.ksplit == 1) {
#pragma unroll
            for (int w = 1; w < kWaves; ++w) sum += red[w][e >> 6][l];
        }
        const int have = min(4, p.N - n);
        if (p.bias) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < have) sum[i] += out_bits_to_f32<kBf16>(p.bias[n + i]);
        }
        const uint32_t o[2] = {mx_round_pair<kBf16>(sum[0], sum[1]), mx_round_pair<kBf16>(sum[2], sum[3])};
        uint16_t* c = p.c + static_cast<int64_t>(m) * p.N + n;
        if (have == 4) {
            __builtin_memcpy(c, o, 8);
        } else {
            for (int i = 0; i < have; ++i) c[i] = static_cast<uint16_t>(o[i >> 1] >> (16 * (i & 1)));
        }
    }
}

template <int MT, int NT>
void launch(const RowsArgs& a, int a_type, bool bf16, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(a.strips * a.ksplit);
    auto go = [&](auto at) {
        if (bf16) mx_rows_kernel<MT, NT, at, true><<<grid, 64 * kWaves, 0, stream>>>(a);
        else mx_rows_kernel<MT, NT, at, false><<<grid, 64 * kWaves, 0, stream>>>(a);
    };
    if (a_type == kMxPacked) go(std::integral_constant<int, kMxPacked>{});
    else if (a_type == kMxBf16) go(std::integral_constant<int, kMxBf16>{});
    else go(std::integral_constant<int, kMxF16>{});
}

// Column tiles of a strip, and workgroups that share one's K steps.
struct RowsPlan {
    int nt;
    int64_t strips, ksplit;
    size_t ws_bytes;
};

// Strips as narrow as one round of workgroups allows, up to four tiles (us with one row and the weight
// in HBM: N=5120 K=5120 in strips of 16 / 32 / 64 columns 9.5 / 7.0 / 8.5, N=13824 16.2 / 11.9 / 10.1,
// N=K=4096 with 16 rows 5.9 / 6.0 / 6.8); K split where strips leave half of the CUs idle and every
// wave keeps two steps (N=512 K=14336 9.6 -> 7.0 in four).
RowsPlan rows_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t ksteps = mx_ksteps(K), tiles = (N + 15) / 16;
    RowsPlan p;
    p.nt = 1;
    while (p.nt < 4 && (tiles + p.nt - 1) / p.nt > 256) p.nt *= 2;
    p.strips = (tiles + p.nt - 1) / p.nt;
    p.ksplit = std::max<int64_t>(1, std::min<int64_t>(128 / p.strips, ksteps / (2 * kWaves)));
    p.ws_bytes = p.ksplit > 1 ? kMxCounterBytes + static_cast<size_t>(p.strips * p.ksplit * p.nt) * (M <= 16 ? 1024 : 2048) : 0;
    return p;
}

}  // namespace

size_t mx_rows_workspace(int64_t M, int64_t N, int64_t K) { return rows_plan(M, N, K).ws_bytes; }

void mx_rows_parts(int64_t M, int64_t N, int64_t K, int64_t* plan) {
    const RowsPlan p = rows_plan(M, N, K);
    plan[0] = M <= 16 ? 16 : 32;
    plan[1] = p.nt * 16;
    plan[2] = p.ksplit;
}

int mx_mm_rows(const MxMmArgs& p, hipStream_t stream) {
    if (p.a_type != kMxPacked && !mx_rows_in_reach(p.M, p.a_stride)) return FEATHER_ERR_UNSUPPORTED;
    RowsPlan plan = rows_plan(p.M, p.N, p.K);
    if (plan.ws_bytes > p.ws_bytes) plan.ksplit = 1;
    const RowsArgs a{p.a, p.a_scales, p.M > 1 ? static_cast<int>(p.a_stride * 2) : 0, p.b, p.b_scales, p.bias, p.c,
                     static_cast<int>(p.M), p.N, p.K, static_cast<int>(mx_ksteps(p.K)), static_cast<int>(plan.strips),
                     static_cast<int>(plan.ksplit), reinterpret_cast<uint32_t*>(p.ws),
                     reinterpret_cast<float*>(p.ws + kMxCounterBytes)};
    auto by_strip = [&](auto mt) {
        if (plan.nt == 4) launch<mt, 4>(a, p.a_type, p.out_bf16, stream);
        else if (plan.nt == 2) launch<mt, 2>(a, p.a_type, p.out_bf16, stream);
        else launch<mt, 1>(a, p.a_type, p.out_bf16, stream);
    };
    if (p.M <= 16) by_strip(std::integral_constant<int, 1>{});
    else by_strip(std::integral_constant<int, 2>{});
    return hipGetLastError() == hipSuccess ? FEATHER_OK : FEATHER_ERR_LAUNCH;
}

}  // namespace feather
