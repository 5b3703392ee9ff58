// The norms around a transformer block in one pass over the residual stream:
//   h' = post_weight ? norm(h) * post_weight : h
//   s  = residual_scale * x + gate * h'          (x where there is no h)
//   y  = norm(s) * weight + bias,  y * (1 + scale) + shift
// with norm(v) = v / sqrt(mean(v^2) + eps) or (v - mean) / sqrt(var + eps). s is kept
// in fp32 from the sum to the norm and rounded once, to the stream's type, on its
// way out; y is rounded once, to 16 bits, or quantised to MXFP4 in the operand order of
// the product that reads it, which saves that product's input a trip to HBM.
//
// HBM bound: x and h are read once and stay in registers (8 values a vector, V
// vectors a thread) over the reductions; the variance is a second sum over the centred
// registers, so a large mean costs no digits. A workgroup owns a row; rows of up to
// 512 values are one wave's, four to a workgroup, and meet no barrier. Measured, with gate, scale
// and shift: 8192 x 5120 with an fp32 stream 99 us (5.1 TB/s; a copy runs at 4.5 to 4.8), 4096 x 5120 in
// bf16 33.5 us (5.0 TB/s), with MXFP4 out 27.6 us (5.1), one row of 5120 3.1 us.
#include <algorithm>
#include <type_traits>

#include "block_norm.h"
#include "featherops_amd.h"
#include "mxfp4.h"

namespace feather {
namespace {

// ---- 8 consecutive values: raw as loaded, and as fp32 ----
template <bool kF32>
struct Raw8 {
    uint4 v[kF32 ? 2 : 1];
};

template <bool kF32>
__device__ __forceinline__ Raw8<kF32> load8(const uint8_t* p) {
    Raw8<kF32> r;
    r.v[0] = load16_unaligned(p);
    if constexpr (kF32) r.v[1] = load16_unaligned(p + 16);
    return r;
}
// values [0, n) of p, zeros beyond
template <bool kF32>
__device__ __forceinline__ Raw8<kF32> load_part(const uint8_t* p, int n) {
    uint32_t w[kF32 ? 8 : 4];
    load_few8<kF32>(p, n, w);
    Raw8<kF32> r;
    r.v[0] = make_uint4(w[0], w[1], w[2], w[3]);
    if constexpr (kF32) r.v[1] = make_uint4(w[4], w[5], w[6], w[7]);
    return r;
}

template <int T>
__device__ __forceinline__ void widen8(const Raw8<T == kMxF32>& r, float (&f)[8]) {
    const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
    if constexpr (T == kMxF32) {
        const uint32_t u[4] = {r.v[1].x, r.v[1].y, r.v[1].z, r.v[1].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = bits_f32(w[i]), f[4 + i] = bits_f32(u[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = out_bits_to_f32<T == kMxBf16>(static_cast<uint16_t>(w[i] & 0xffffu));
            f[2 * i + 1] = out_bits_to_f32<T == kMxBf16>(static_cast<uint16_t>(w[i] >> 16));
        }
    }
}

// kTiny: the first n values
template <int T, bool kTiny>
__device__ __forceinline__ void store8(uint8_t* p, const float (&f)[8], int n) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (T == kMxF32) w[i] = f32_bits(f[i]);
        else if (i < 4) w[i] = mx_round_pair<T == kMxBf16>(f[2 * i], f[2 * i + 1]);
    }
    if constexpr (!kTiny) {
        __builtin_memcpy(p, w, T == kMxF32 ? 32 : 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= n) continue;
            if constexpr (T == kMxF32) reinterpret_cast<uint32_t*>(p)[i] = w[i];
            else reinterpret_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
        }
    }
}

// ---- sums ----
template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
    return bits_f32(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(f32_bits(v)), kCtrl, 0xf, 0xf, true)));
}
__device__ __forceinline__ float sum16(float v) {
    v += dpp<0xB1>(v);   // lane ^ 1
    v += dpp<0x4E>(v);   // lane ^ 2
    v += dpp<0x141>(v);  // the other four of eight
    v += dpp<0x140>(v);  // the other eight of sixteen
    return v;
}
__device__ __forceinline__ float sum64(float v) {
    v = sum16(v);
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    return v;
}

// The sum over a row's threads, the same bits in each of them: waves' sums are added in
// lane order. buf: 16 floats of its own for each call.
template <bool kOneWave>
__device__ __forceinline__ float row_sum(float v, float* buf, int waves) {
    v = sum64(v);
    if constexpr (kOneWave) return v;
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    const int l = threadIdx.x & 15;
    return sum16(l < waves ? buf[l] : 0.f);
}

template <int T>
constexpr int kBytes = T == kMxF32 ? 4 : 2;

// TX: the stream's type, TY: the block's, kModF32: the vectors' (else TY), V: vectors a thread.
// A row's last vector, where its width is no multiple of 8, is moved back to end with the row: it repeats
// values of the vector before it, which stay out of the sums and are stored twice, the same both times.
// So no load has a partial form, whose branch would make each load wait for the one before.
// kTiny: rows of fewer than 8 values.
template <int TX, int TY, bool kModF32, int V, bool kOneWave, bool kCodes, bool kTiny>
// (one vector a thread: 64 registers, so that a CU holds three workgroups of ten waves)
__global__ __launch_bounds__(kOneWave ? 256 : 1024, V == 1 ? 8 : 4) void norm_kernel(const NormArgs p, int ksteps) {
    constexpr int TM = kModF32 ? kMxF32 : TY;
    __shared__ float sums[4][16];
    const int threads = kOneWave ? 64 : blockDim.x;
    const int tid = kOneWave ? threadIdx.x & 63 : threadIdx.x;
    const int waves = threads >> 6;
    int64_t row;
    if constexpr (kCodes && !kOneWave) {
        // 16 rows fill the packed operand's cache lines together: they go to one XCD (workgroup
        // p runs on XCD p % 8), whose L2 gathers their pieces
        const int64_t b = blockIdx.x;
        row = (b / 128 * 8 + b % 8) * 16 + b / 8 % 16;
    } else {
        row = kOneWave ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6) : blockIdx.x;
    }
    row += p.row0;
    if (row >= p.rows) return;  // (whole rows: no thread of a row that takes part leaves)

    // vector i of this thread: the columns it stands for, where it lies, and how many of its values another
    // vector stands for (8 or more: all of them, a vector past the row's end)
    auto at = [&](int i) { return (tid + i * threads) * 8; };
    auto lies = [&](int i) { return kTiny ? at(i) : min(at(i), p.cols - 8); };
    auto shared_values = [&](int i) { return at(i) - lies(i); };
    auto vec = [&](const void* base, int64_t offset, int i, auto f32) {
        const uint8_t* v = static_cast<const uint8_t*>(base) + (offset + lies(i)) * (f32 ? 4 : 2);
        if constexpr (kTiny) return load_part<f32>(v, p.cols - at(i));
        else return load8<f32>(v);
    };
    // the sum of f over the values that this thread's vectors stand for
    auto sum_of = [&](const float (&v)[V][8], auto f) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float part = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) part += f(v[i][e]);
            const int skip = shared_values(i);
            if (kTiny || skip > 0) {
                part = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e >= skip && (!kTiny || at(i) + e < p.cols)) part += f(v[i][e]);
            }
            s += part;
        }
        return s;
    };
    typedef std::integral_constant<bool, TX == kMxF32> XF;
    typedef std::integral_constant<bool, TY == kMxF32> YF;
    typedef std::integral_constant<bool, TM == kMxF32> MF;

    Raw8<TX == kMxF32> xr[V];
    Raw8<TY == kMxF32> hr[V];
    Raw8<TM == kMxF32> gr[V], pr[V];
#pragma unroll
    for (int i = 0; i < V; ++i) xr[i] = vec(p.x, row * p.x_stride, i, XF{});
    if (p.h) {
#pragma unroll
        for (int i = 0; i < V; ++i) hr[i] = vec(p.h, row * p.h_stride, i, YF{});
        if (p.post_weight) {
#pragma unroll
            for (int i = 0; i < V; ++i) pr[i] = vec(p.post_weight, 0, i, MF{});
        }
        if (p.gate) {
            const int64_t g = (static_cast<uint32_t>(row) / p.gate_group) * p.gate_stride;
#pragma unroll
            for (int i = 0; i < V; ++i) gr[i] = vec(p.gate, g, i, MF{});
        }
    }
    // divided, not multiplied by a rounded reciprocal: a row of equal values has exactly that mean
    const float count = static_cast<float>(p.cols);
    auto normalise = [&](float (&v)[V][8], float* buf) {
        if (p.layer) {
            const float mean = row_sum<kOneWave>(sum_of(v, [](float a) { return a; }), buf, waves) / count;
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] -= mean;
        }
        const float r = 1.0f / sqrtf(row_sum<kOneWave>(sum_of(v, [](float a) { return a * a; }), buf + 16, waves) / count + p.eps);
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] *= r;
    };

    float s[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i) widen8<TX>(xr[i], s[i]);
    if (p.h) {
        float h[V][8];
#pragma unroll
        for (int i = 0; i < V; ++i) widen8<TY>(hr[i], h[i]);
        if (p.post_weight) {
            normalise(h, sums[0]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float w[8];
                widen8<TM>(pr[i], w);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[i][e] *= w[e];
            }
        }
        if (p.residual_scale != 1.0f) {
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[i][e] *= p.residual_scale;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (p.gate) {
                float g[8];
                widen8<TM>(gr[i], g);
#pragma unroll
                for (int e = 0; e < 8; ++e) s[i][e] = fmaf(h[i][e], g[e], s[i][e]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) s[i][e] += h[i][e];
            }
            if (at(i) < p.cols)
                store8<TX, kTiny>(static_cast<uint8_t*>(p.x_out) + (row * p.cols + lies(i)) * kBytes<TX>, s[i], p.cols - at(i));
        }
    }
    // the affine vectors travel while the reductions run
    Raw8<TM == kMxF32> wr[V], br[V], sr[V], tr[V];
    if (p.weight) {
#pragma unroll
        for (int i = 0; i < V; ++i) wr[i] = vec(p.weight, 0, i, MF{});
    }
    if (p.bias) {
#pragma unroll
        for (int i = 0; i < V; ++i) br[i] = vec(p.bias, 0, i, MF{});
    }
    const int64_t mod_row = (p.scale || p.shift) ? static_cast<uint32_t>(row) / p.mod_group : 0;
    if (p.scale) {
#pragma unroll
        for (int i = 0; i < V; ++i) sr[i] = vec(p.scale, mod_row * p.scale_stride, i, MF{});
    }
    if (p.shift) {
#pragma unroll
        for (int i = 0; i < V; ++i) tr[i] = vec(p.shift, mod_row * p.shift_stride, i, MF{});
    }
    normalise(s, sums[2]);
    // (this row's place in the packed operand; the columns' place in it is the thread's)
    uint8_t* row_codes = kCodes ? p.codes + ((row >> 6) * ksteps * 4 + ((row >> 4) & 3)) * 1024 + (row & 15) * 16 : nullptr;
    uint8_t* row_scales = kCodes ? p.scales + (row >> 6) * ksteps * 256 + (row & 15) * 4 + ((row >> 4) & 3) : nullptr;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float (&y)[8] = s[i];
        float t[8];
        if (p.weight) {
            widen8<TM>(wr[i], t);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] *= t[e];
        }
        if (p.bias) {
            widen8<TM>(br[i], t);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] += t[e];
        }
        if (p.scale) {
            widen8<TM>(sr[i], t);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] *= 1.0f + t[e];
        }
        if (p.shift) {
            widen8<TM>(tr[i], t);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] += t[e];
        }
        const int c = at(i);
        if constexpr (!kCodes) {
            if (c < p.cols) store8<TY, kTiny>(static_cast<uint8_t*>(p.y) + (row * p.cols + lies(i)) * kBytes<TY>, y, p.cols - c);
        } else {
            // four neighbouring lanes hold a block of 32 (columns beyond the row are zeros in y's place)
            if (kTiny || c + 8 > p.cols) {  // columns in their own places, zeros beyond the row
                const int skip = shared_values(i);
#pragma unroll
                for (int by = 4; by >= 1; by /= 2) {
                    if (skip & by) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = e + by < 8 ? y[e + by] : 0.f;
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e >= p.cols) y[e] = 0.f;
            }
            uint32_t m = 0u;
#pragma unroll
            for (int e = 0; e < 8; ++e) m = max(m, f32_bits(y[e]) & 0x7fffffffu);
            m = max(m, quad_perm<kQuadXor1>(m));
            m = max(m, quad_perm<kQuadXor2>(m));
            const uint32_t sb = mx_scale_byte(bits_f32(m));
            const float q = mx_scale_f32(sb);
            uint32_t o = 0u;
            o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, y[0], y[1], q, 0);
            o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, y[2], y[3], q, 1);
            o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, y[4], y[5], q, 2);
            o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, y[6], y[7], q, 3);
            if (c < ksteps * kMxStepK) {
                *reinterpret_cast<uint32_t*>(row_codes + c / kMxStepK * 4096 + c % kMxStepK / kMxBlock * 256 + c % kMxBlock / 2) = o;
                if (c % kMxBlock == 0) row_scales[c / kMxBlock * 64] = static_cast<uint8_t>(sb);
            }
        }
    }
}

// Rows of one launch: a grid holds fewer than 2^32 threads, and a row takes up to 1024.
constexpr int64_t kLaunchRows = int64_t(1) << 21;

// Rows [p.row0, p.row0 + rows).
template <int TX, int TY, bool kModF32, int V>
int launch_rows(const NormArgs& p, int64_t rows, int threads, hipStream_t stream) {
    const int ksteps = static_cast<int>(mx_ksteps(p.cols));
    typedef std::integral_constant<bool, true> Yes;
    typedef std::integral_constant<bool, false> No;
    auto go = [&](auto one_wave, auto codes, auto tiny, int64_t blocks, int block_threads) {
        norm_kernel<TX, TY, kModF32, V, one_wave, codes, tiny>
            <<<static_cast<unsigned>(blocks), block_threads, 0, stream>>>(p, ksteps);
    };
    bool one_wave = false;
    if constexpr (V == 1) {  // (two vectors a thread: only rows of five waves or more, see pick)
        one_wave = threads == 64;
        if (one_wave) {
            const int64_t blocks = (rows + 3) / 4;
            if (p.cols < 8) {
                if (p.codes) go(Yes{}, Yes{}, Yes{}, blocks, 256);
                else go(Yes{}, No{}, Yes{}, blocks, 256);
            } else {
                if (p.codes) go(Yes{}, Yes{}, No{}, blocks, 256);
                else go(Yes{}, No{}, No{}, blocks, 256);
            }
        }
    }
    if (!one_wave) {
        if (p.codes) go(No{}, Yes{}, No{}, (rows + 127) / 128 * 128, threads);  // whole rounds of 16 rows on each XCD
        else go(No{}, No{}, No{}, rows, threads);
    }
    return hipGetLastError() == hipSuccess ? FEATHER_OK : FEATHER_ERR_LAUNCH;
}

template <int TX, int TY, bool kModF32, int V>
int launch(NormArgs p, int threads, hipStream_t stream) {
    int st = FEATHER_OK;
    for (p.row0 = 0; p.row0 < p.rows && st == FEATHER_OK; p.row0 += kLaunchRows)
        st = launch_rows<TX, TY, kModF32, V>(p, std::min(kLaunchRows, p.rows - p.row0), threads, stream);
    return st;
}

template <int TX, int TY, bool kModF32>
int pick(const NormArgs& p, hipStream_t stream) {
    const int64_t cols = p.codes ? mx_ksteps(p.cols) * kMxStepK : p.cols;
    const int64_t vecs = (cols + 7) / 8;
    auto threads = [&](int n) { return static_cast<int>((vecs + 64 * n - 1) / (64 * n) * 64); };
    // One vector a thread where that keeps the workgroup to 512 threads, for an fp32 stream (32 bytes a vector
    // already; 8192 x 5120: 97 against 109 us) and for few rows, whose latency shows (one row of 5120: 4.1
    // against 4.5 us); otherwise two (4096 x 5120 in bf16: 35 against 41 us).
    return threads(1) <= 512 || (threads(1) <= 1024 && (TX == kMxF32 || p.rows <= 1024))
               ? launch<TX, TY, kModF32, 1>(p, threads(1), stream)
               : launch<TX, TY, kModF32, 2>(p, threads(2), stream);
}

}  // namespace

int block_norm(const NormArgs& p, hipStream_t stream) {
    if (p.x_type == kMxF32) {
        if (p.y_type == kMxF32) return pick<kMxF32, kMxF32, true>(p, stream);
        if (p.y_type == kMxBf16) return p.mod_f32 ? pick<kMxF32, kMxBf16, true>(p, stream) : pick<kMxF32, kMxBf16, false>(p, stream);
        return p.mod_f32 ? pick<kMxF32, kMxF16, true>(p, stream) : pick<kMxF32, kMxF16, false>(p, stream);
    }
    if (p.x_type == kMxBf16) return p.mod_f32 ? pick<kMxBf16, kMxBf16, true>(p, stream) : pick<kMxBf16, kMxBf16, false>(p, stream);
    return p.mod_f32 ? pick<kMxF16, kMxF16, true>(p, stream) : pick<kMxF16, kMxF16, false>(p, stream);
}

}  // namespace feather
