// Rotary positions of several axes, and the norm of queries and keys that comes before them:
//   v = x / sqrt(mean(x^2) + eps) * weight     over a head, over all heads of a token, or left out
//   (a, b) -> (a cos - b sin, b cos + a sin)   for each pair of a head's values
// A pair is two adjacent values, or one value of the first and one of the second half of the values that turn; values
// behind them stay. Everything is fp32 from the input to the one rounding of the result.
//
// The table of cosines and sines holds fp32 pairs, computed from angles in fp64: a position of
// 100000 has 17 bits before the point, and an fp32 angle would keep 7 behind it.
//
// HBM bound: x is read once and stays in registers over the norm. 32760 tokens x 40 heads of 128 with a norm of the row:
// 250 us, 5.4 TB/s (a 1 GiB copy: 5.1); 2 x 4250 x 24 heads with one of the head 37 us of kernel. A lane has 8 values of a head; a wave takes
// one token's heads, several in a row, so that the table's values are loaded once for them. With pairs of
// two halves the partner's values come through LDS. Where the norm is over all heads a workgroup has
// the token.
#include <algorithm>

#include "feather_common.h"
#include "lds_dma.h"
#include "featherops_amd.h"
#include "mxfp4.h"
#include "rope.h"

namespace feather {
namespace {

constexpr int kThreads = 256;

template <int T>
constexpr int kSize = T == kMxF32 ? 4 : 2;

template <int T>
struct Values8 {
    uint4 w[T == kMxF32 ? 2 : 1];
};
template <int T>
__device__ __forceinline__ Values8<T> load8(const uint8_t* p) {
    Values8<T> v;
    v.w[0] = load16_unaligned(p);
    if constexpr (T == kMxF32) v.w[1] = load16_unaligned(p + 16);
    return v;
}
template <int T>
__device__ __forceinline__ void widen8(const Values8<T>& v, float (&f)[8]) {
    if constexpr (T == kMxF32) {
        __builtin_memcpy(f, v.w, 32);
    } else {
        const uint32_t w[4] = {v.w[0].x, v.w[0].y, v.w[0].z, v.w[0].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = out_bits_to_f32<T == kMxBf16>(static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2))));
    }
}
template <int T>
__device__ __forceinline__ void store8(uint8_t* p, const float (&f)[8]) {
    if constexpr (T == kMxF32) {
        __builtin_memcpy(p, f, 32);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == kMxBf16) w[i] = f32x2_to_bf16x2_raw(f[2 * i], f[2 * i + 1]);
            else w[i] = f32x2_to_out_bits<false>(f[2 * i], f[2 * i + 1]);
        }
        __builtin_memcpy(p, w, 16);
    }
}

// The sum over each `lanes` lanes (a power of two), in all of them.
template <int kControl>
__device__ __forceinline__ float add_lane(float x) {
    return x + bits_f32(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(f32_bits(x)), kControl, 0xf, 0xf, true)));
}
__device__ __forceinline__ float sum_lanes(float x, int lanes) {
    if (lanes > 1) x = add_lane<0xB1>(x);   // the neighbour's
    if (lanes > 2) x = add_lane<0x4E>(x);   // the other pair's of four
    if (lanes > 4) x = add_lane<0x141>(x);  // mirrored in eight, whose fours are alike by now
    if (lanes > 8) x = add_lane<0x140>(x);  // and in sixteen
    if (lanes > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(f32_bits(x), f32_bits(x), false, false);
        x = bits_f32(r[0]) + bits_f32(r[1]);
    }
    if (lanes > 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(f32_bits(x), f32_bits(x), false, false);
        x = bits_f32(r[0]) + bits_f32(r[1]);
    }
    return x;
}

// The eight values of a lane in LDS, in two planes of four so that neighbours' 16 bytes lie next to each other.
struct Plane {
    float4 quad[2][64];
};

// kPasses: heads of a lane. A pass has 64 / lanes heads, or 256 / lanes where the norm is over the row.
// kPartly: a part of a head turns, and the values behind it are left alone: times 1 and plus a neighbour times 0 would make NaN
// of infinities. (Asked of heads that turn as a whole, too, it took 259 us for 252 at 32760 tokens x 40 + 40 heads.)
template <int T, int kPasses, bool kRow, bool kPartly>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(const RopeArgs p, int lanes, uint32_t items, uint32_t chunks_q,
                                                                uint32_t chunks) {
    __shared__ Plane planes[kThreads / 64];
    __shared__ float sums[kThreads / 64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int slot = kRow ? threadIdx.x : lane;
    const int heads_a_pass = (kRow ? kThreads : 64) / lanes;
    const int head_in_pass = slot / lanes, d = slot % lanes * 8;
    const bool has = d < p.dim;
    Plane& plane = planes[wave];

    const uint32_t item = kRow ? blockIdx.x : blockIdx.x * (kThreads / 64) + wave;
    if (item >= items) return;
    const uint32_t token = item / chunks, chunk = item - token * chunks;
    const bool of_keys = chunk >= chunks_q;
    const RopeSide& side = p.side[of_keys];
    const uint32_t b = token / static_cast<uint32_t>(p.per_sample), s = token - b * p.per_sample;
    const int head0 = (chunk - (of_keys ? chunks_q : 0)) * heads_a_pass * kPasses + head_in_pass;
    const uint8_t* x = side.x + b * side.batch_stride + s * side.token_stride + d * kSize<T>;

    Values8<T> raw[kPasses];
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        const int head = head0 + u * heads_a_pass;
        raw[u] = {};
        if (has && head < side.heads) raw[u] = load8<T>(x + head * side.head_stride);
    }
    // weights: one for all heads, or with a norm over the row each head's
    constexpr int kWeights = kRow ? kPasses : 1;
    Values8<kMxF32> weight[kWeights];
    if (side.weight && has) {
#pragma unroll
        for (int u = 0; u < kWeights; ++u) {
            const int head = kRow ? head0 + u * heads_a_pass : 0, at = head * p.dim + d;
            if (head >= side.heads) continue;
            const uint8_t* from = static_cast<const uint8_t*>(side.weight);
            if (p.weight_f32) weight[u] = load8<kMxF32>(from + at * 4);
            else weight[u].w[0] = load8<T>(from + at * kSize<T>).w[0];  // (fp32 values have fp32 weights)
        }
    }
    // the turn of each value: its pair's cosine and, with the sign of its place in the pair, sine
    float cosine[8], sine[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) cosine[i] = 1.0f, sine[i] = 0.0f;
    const int turned = 2 * p.pairs;
    if (p.table && d < turned) {
        const float* row = p.table + b * p.table_batch + static_cast<int64_t>(s) * turned;
        if (!p.halves) {
            float t[8];
            if (d + 8 <= turned) {
                __builtin_memcpy(t, row + d, 32);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = d + i < turned ? row[d + i] : i % 2 ? 0.0f : 1.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                cosine[i] = cosine[i + 1] = t[i];
                sine[i] = -t[i + 1];
                sine[i + 1] = t[i + 1];
            }
        } else if (p.pairs % 8 == 0) {
            const bool second = d >= p.pairs;
            float t[16];
            __builtin_memcpy(t, row + (second ? d - p.pairs : d) * 2, 64);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                cosine[i] = t[2 * i];
                sine[i] = second ? t[2 * i + 1] : -t[2 * i + 1];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = d + i;
                if (e < turned) {
                    const float* t = row + (e < p.pairs ? e : e - p.pairs) * 2;
                    cosine[i] = t[0];
                    sine[i] = e < p.pairs ? -t[1] : t[1];
                }
            }
        }
    }

    float v[kPasses][8], square[kPasses];
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        widen8<T>(raw[u], v[u]);
        square[u] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) square[u] += v[u][i] * v[u][i];
    }
    if (kRow) {
        float all = 0.0f;
#pragma unroll
        for (int u = 0; u < kPasses; ++u) all += square[u];
        all = sum_lanes(all, 64);
        if (lane == 0) sums[wave] = all;
        __syncthreads();
        all = 0.0f;
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) all += sums[w];
        const float by = 1.0f / __builtin_sqrtf(all / (static_cast<float>(side.heads) * p.dim) + p.eps);
#pragma unroll
        for (int u = 0; u < kPasses; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] *= by;
    } else if (p.norm) {
        const float one = 1.0f / p.dim;
#pragma unroll
        for (int u = 0; u < kPasses; ++u) {
            const float by = __builtin_amdgcn_rsqf(sum_lanes(square[u], lanes) * one + p.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] *= by;
        }
    }
    if (side.weight) {
#pragma unroll
        for (int u = 0; u < kPasses; ++u) {
            float f[8];
            if (p.weight_f32) {
                widen8<kMxF32>(weight[kRow ? u : 0], f);
            } else {
                Values8<T> h{};
                h.w[0] = weight[kRow ? u : 0].w[0];
                widen8<T>(h, f);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] *= f[i];
        }
    }

    uint8_t* out = side.out + static_cast<int64_t>(token) * side.heads * p.dim * kSize<T> + d * kSize<T>;
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        const int head = head0 + u * heads_a_pass;
        if (p.table) {
            float other[8];
            if (p.halves) {
                plane.quad[0][lane] = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
                plane.quad[1][lane] = make_float4(v[u][4], v[u][5], v[u][6], v[u][7]);
                wave_lds_sync();
                const int first = lane / lanes * lanes;  // the lane with the head's first values
                if (p.pairs % 4 == 0) {
                    // four values at once have their partners next to each other, on one side
#pragma unroll
                    for (int i = 0; i < 8; i += 4) {
                        const int e = d + i, from = e < p.pairs ? e + p.pairs : e < turned ? e - p.pairs : e;
                        const float4 q = plane.quad[from / 4 % 2][(first + from / 8) % 64];
                        other[i] = q.x, other[i + 1] = q.y, other[i + 2] = q.z, other[i + 3] = q.w;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int e = d + i, from = e < p.pairs ? e + p.pairs : e < turned ? e - p.pairs : e;
                        other[i] = reinterpret_cast<const float*>(&plane.quad[from / 4 % 2][(first + from / 8) % 64])[from % 4];
                    }
                }
                wave_lds_sync();  // (read before the next pass writes)
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) other[i] = v[u][i ^ 1];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!kPartly || d + i < turned) v[u][i] = v[u][i] * cosine[i] + other[i] * sine[i];
        }
        if (has && head < side.heads) store8<T>(out + static_cast<int64_t>(head) * p.dim * kSize<T>, v[u]);
    }
}

template <int T, int kPasses, bool kRow>
int launch(const RopeArgs& p, int lanes, hipStream_t stream) {
    const int heads = (kRow ? kThreads : 64) / lanes * kPasses;
    const int chunks_q = (p.side[0].heads + heads - 1) / heads, chunks = chunks_q + (p.side[1].heads + heads - 1) / heads;
    const int64_t items = p.tokens * chunks, blocks = kRow ? items : (items + kThreads / 64 - 1) / (kThreads / 64);
    if (blocks * kThreads > 0xffffffffll) return FEATHER_ERR_UNSUPPORTED;  // (2^24 workgroups)
    auto* kernel = p.table && 2 * p.pairs < p.dim ? qk_norm_rope_kernel<T, kPasses, kRow, true> : qk_norm_rope_kernel<T, kPasses, kRow, false>;
    kernel<<<dim3(static_cast<uint32_t>(blocks)), kThreads, 0, stream>>>(p, lanes, static_cast<uint32_t>(items), chunks_q, chunks);
    return hipGetLastError() == hipSuccess ? FEATHER_OK : FEATHER_ERR_LAUNCH;
}

template <int T>
int of_type(const RopeArgs& p, hipStream_t stream) {
    int lanes = 1;
    while (lanes * 8 < p.dim) lanes *= 2;
    const int most = std::max(p.side[0].heads, p.side[1].heads);
    if (p.norm == kNormRow) {
        const int passes = (most * lanes + kThreads - 1) / kThreads;
        if (passes <= 1) return launch<T, 1, true>(p, lanes, stream);
        if (passes <= 2) return launch<T, 2, true>(p, lanes, stream);
        if (passes <= 3) return launch<T, 3, true>(p, lanes, stream);
        if (passes <= 4) return launch<T, 4, true>(p, lanes, stream);
        return launch<T, 8, true>(p, lanes, stream);
    }
    // Few tokens: a wave for every 64 / lanes heads (100 tokens of 24 heads of 128: 4.0 us, with two passes 4.1). Many: two passes,
    // for which the table is loaded once (20000 tokens of 24 heads of 96: 89 us with one pass, 70 with two). Three and four
    // leave too few waves, or their last pass idle (65536 tokens of 32 + 4 heads of 128 221 us with two, 241 and 238;
    // 3 x 1003 of 15 + 15 of 80 12.4, 15.1 and 12.5; only of 32760 x 40 + 40 three are 2% faster).
    const int all = (most * lanes + 63) / 64;
    return p.tokens < 256 || all <= 1 ? launch<T, 1, false>(p, lanes, stream) : launch<T, 2, false>(p, lanes, stream);
}

__global__ __launch_bounds__(kThreads) void rope_table_kernel(const RopeTableArgs p) {
    const int64_t n = p.rows * p.pairs, step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += step) {
        const int64_t row = i / p.pairs;
        const int pair = static_cast<int>(i - row * p.pairs);
        int axis = 0;
        while (pair >= p.first[axis + 1]) ++axis;
        const int64_t at = row * p.axes + axis;
        double position;
        switch (p.position_type) {
            case 0: position = static_cast<const int*>(p.positions)[at]; break;
            case 1: position = static_cast<double>(static_cast<const int64_t*>(p.positions)[at]); break;
            case 2: position = static_cast<const float*>(p.positions)[at]; break;
            default: position = static_cast<const double*>(p.positions)[at];
        }
        // pair j of an axis of d values (or of all of them) turns by theta^(-2 j / d); in half turns, whose
        // sine and cosine need no reduction by pi
        const int of = p.shared ? p.pairs : p.first[axis + 1] - p.first[axis];
        const int j = p.shared ? pair : pair - p.first[axis];
        const double half_turns = position * (exp(-p.log_theta * j / of) * 0.31830988618379067);
        double sine, cosine;
        sincospi(half_turns, &sine, &cosine);
        reinterpret_cast<float2*>(p.table)[i] = make_float2(static_cast<float>(cosine), static_cast<float>(sine));
    }
}

}  // namespace

int qk_norm_rope(const RopeArgs& p, hipStream_t stream) {
    switch (p.type) {
        case FEATHER_DTYPE_F16: return of_type<kMxF16>(p, stream);
        case FEATHER_DTYPE_BF16: return of_type<kMxBf16>(p, stream);
        default: return of_type<kMxF32>(p, stream);
    }
}

int rope_table(const RopeTableArgs& p, hipStream_t stream) {
    const int64_t blocks = (p.rows * p.pairs + kThreads - 1) / kThreads;
    rope_table_kernel<<<dim3(static_cast<uint32_t>(std::min<int64_t>(blocks, 1 << 14))), kThreads, 0, stream>>>(p);
    return hipGetLastError() == hipSuccess ? FEATHER_OK : FEATHER_ERR_LAUNCH;
}

}  // namespace feather
