// The MXFP4 product for few rows: C (M, N) = q(A) . B^T + bias, where the call is
// bound by streaming the weight once. 16-bit activations are quantised on the way
// into the matrix instruction: lane l of the operand holds one block of 32 values of
// row l % 16, so its scale and codes need no other lane and cost ~50 instructions
// beside the 2 KB or more of weights the wave waits for; a launch of its own for
// the quantisation would cost more than the whole product of one token.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "featherops_amd.h"
#include "mxfp4.h"

namespace feather {
namespace {

constexpr int kWaves = 8;

template <int... I, class F>
__device__ __forceinline__ void unrolled_impl(std::integer_sequence<int, I...>, F&& f) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void unrolled(F&& f) {
    unrolled_impl(std::make_integer_sequence<int, N>{}, f);
}

struct RowsArgs {
    const uint8_t* a;
    const uint8_t* as;
    int64_t a_row_bytes;
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
    std::conditional_t<AT == kMxPacked, uint4, MxRaw<AT == kMxBf16 ? kMxBf16 : kMxF16>> a[MT];
    uint32_t as, bs;
    uint4 b[NT];
};

// A workgroup takes NT column tiles (a strip) and all MT row tiles; its waves take
// the K steps in turn, kDepth steps' loads in flight each, and add their sums
// through LDS in wave order. ksplit > 1: several workgroups share a strip's steps.
template <int MT, int NT, int AT, bool kBf16>
__global__ __launch_bounds__(64 * kWaves) void mx_rows_kernel(const RowsArgs p) {
    constexpr int kDepth = 3;
    __shared__ __attribute__((aligned(16))) f32x4 red[kWaves][MT * NT][64];
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int lr = lane & 15;
    const int kb = lane >> 4;

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
    const uint8_t* b = p.b + tile0 * p.ksteps * 1024 + lane * 16;
    const uint8_t* bs = p.bs + (tile0 / 4) * p.ksteps * 256 + lane * 4;
    const int bshift = 8 * static_cast<int>(tile0 % 4);
    typedef Step<MT, NT, AT> S;
    auto load = [&](S& s, int k) {
        if constexpr (AT == kMxPacked) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
                s.a[i] = *reinterpret_cast<const uint4*>(p.a + (static_cast<int64_t>(i) * p.ksteps + k) * 1024 + lane * 16);
            s.as = *reinterpret_cast<const uint32_t*>(p.as + static_cast<int64_t>(k) * 256 + lane * 4);
        } else {
            const int col = k * kMxStepK + kb * kMxBlock;
            const int n = max(0, min(kMxBlock, p.K - col));
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int row = i * 16 + lr;
                s.a[i].load(p.a + row * p.a_row_bytes + static_cast<int64_t>(col) * 2, row < p.M ? n : 0);
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
            s.b[j] = *reinterpret_cast<const uint4*>(b + (static_cast<int64_t>(j) * p.ksteps + k) * 1024);
        s.bs = *reinterpret_cast<const uint32_t*>(bs + static_cast<int64_t>(k) * 256);
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
                a = s.a[i].quantize(&ascale);
            }
            unrolled<NT>([&](auto j) { acc[i][j] = mfma_mx<j, kByte>(s.b[j], a, acc[i][j], bscale, ascale); });
        });
    };

    S buf[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
        if (k0 + wave + d * kWaves < k1) load(buf[d], k0 + wave + d * kWaves);
    for (int k = k0 + wave; k < k1; k += kDepth * kWaves) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            const int kd = k + d * kWaves;
            if (kd < k1) {
                multiply(buf[d]);
                if (kd + kDepth * kWaves < k1) load(buf[d], kd + kDepth * kWaves);
            }
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
        const uint32_t o[2] = {f32x2_to_out_bits<kBf16>(sum[0], sum[1]), f32x2_to_out_bits<kBf16>(sum[2], sum[3])};
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

}  // namespace

// tile: the strip's column tiles
MxPlan mx_rows_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t ksteps = mx_ksteps(K);
    const int64_t tiles = (N + 15) / 16;
    int nt = 4;
    while (nt > 1 && (tiles + nt - 1) / nt < 256) nt /= 2;
    const int64_t strips = (tiles + nt - 1) / nt;
    int64_t ksplit = 1;
    if (strips < 160) ksplit = std::max<int64_t>(1, std::min<int64_t>(256 / strips, ksteps / kWaves));
    const int64_t mt = (M + 15) / 16;
    size_t ws = 0;
    if (ksplit > 1) ws = kMxCounterBytes + static_cast<size_t>(strips) * ksplit * mt * nt * 1024;
    return {nt, static_cast<int>(ksplit), ws};
}

bool mx_takes_rows(int64_t M, int64_t N, int64_t K, int a_type) { return M <= 16; }

int mx_mm_rows(const MxMmArgs& p, hipStream_t stream) {
    MxPlan plan = mx_rows_plan(p.M, p.N, p.K);
    if (plan.ws_bytes > p.ws_bytes) plan.ksplit = 1;
    const int nt = plan.tile;
    const RowsArgs a{p.a, p.a_scales, p.a_stride * 2, p.b, p.b_scales, p.bias, p.c, static_cast<int>(p.M), p.N, p.K,
                     static_cast<int>(mx_ksteps(p.K)), static_cast<int>(((p.N + 15) / 16 + nt - 1) / nt), plan.ksplit,
                     reinterpret_cast<uint32_t*>(p.ws), reinterpret_cast<float*>(p.ws + kMxCounterBytes)};
    if (nt == 4) launch<1, 4>(a, p.a_type, p.out_bf16, stream);
    else if (nt == 2) launch<1, 2>(a, p.a_type, p.out_bf16, stream);
    else launch<1, 1>(a, p.a_type, p.out_bf16, stream);
    return hipGetLastError() == hipSuccess ? FEATHER_OK : FEATHER_ERR_LAUNCH;
}

}  // namespace feather
