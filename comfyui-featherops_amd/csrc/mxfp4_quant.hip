// MXFP4 quantisation and its layouts: row-major values <-> packed operands, and
// the row-major codes of checkpoints <-> packed operands. Formats in mxfp4.h.
//
// All four kernels give one wave a group of 64 rows and one step of 128 columns:
// lane l has row l % 16 of each of the group's four row tiles and the block of 32
// columns l / 16, the packed layout's own order, so a block's maximum needs no
// other lane, codes leave as whole KBs and the four tiles' scales as one dword
// per lane. The row-major side is read (written) in runs of 256 bytes per row
// (16-bit values). HBM bound.
#include "featherops_amd.h"
#include "mxfp4.h"

namespace feather {
namespace {

constexpr int kWavesPerBlock = 4;

// The wave's group and step: consecutive waves take consecutive steps of a group.
struct WaveTask {
    int64_t group;
    int step, lane, lr, kb;
    bool ok;
    __device__ __forceinline__ WaveTask(int64_t groups, int ksteps) {
        const int64_t w = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + (threadIdx.x >> 6);
        ok = w < groups * ksteps;
        group = w / ksteps;
        step = static_cast<int>(w - group * ksteps);
        lane = threadIdx.x & 63;
        lr = lane & 15;
        kb = lane >> 4;
    }
    __device__ __forceinline__ int64_t row(int f) const { return group * 64 + f * 16 + lr; }
    __device__ __forceinline__ int64_t code_at(int f, int ksteps) const {
        return ((group * 4 + f) * ksteps + step) * 1024 + lane * 16;
    }
    __device__ __forceinline__ int64_t scale_at(int ksteps) const { return (group * ksteps + step) * 256 + lane * 4; }
    // how many of the lane's 32 columns exist
    __device__ __forceinline__ int count(int cols) const {
        const int n = cols - step * kMxStepK - kb * kMxBlock;
        return n < 0 ? 0 : n > kMxBlock ? kMxBlock : n;
    }
};

template <int T>
__global__ __launch_bounds__(64 * kWavesPerBlock) void quantize_kernel(const uint8_t* __restrict__ x, int64_t rows,
                                                                       int cols, int64_t row_bytes,
                                                                       uint8_t* __restrict__ codes,
                                                                       uint8_t* __restrict__ scales, int ksteps,
                                                                       int64_t groups) {
    const WaveTask t(groups, ksteps);
    if (!t.ok) return;
    const int n = t.count(cols);
    MxRaw<T> raw[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const int64_t row = t.row(f);
        const int64_t at = row * row_bytes + (static_cast<int64_t>(t.step) * kMxStepK + t.kb * kMxBlock) * kMxElemBytes<T>;
        raw[f].load(x + at, row < rows ? n : 0);
    }
    uint32_t bytes = 0u;
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        uint32_t s;
        const uint4 q = raw[f].quantize(&s);
        *reinterpret_cast<uint4*>(codes + t.code_at(f, ksteps)) = q;
        bytes |= s << (8 * f);
    }
    *reinterpret_cast<uint32_t*>(scales + t.scale_at(ksteps)) = bytes;
}

// Two codes of byte `byte` of w as fp32, times the scale (NaN under scale 255).
template <int kByte>
__device__ __forceinline__ f32x2_t codes_to_f32(uint32_t w, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, kByte);
}

template <int T>
__global__ __launch_bounds__(64 * kWavesPerBlock) void dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                         const uint8_t* __restrict__ scales,
                                                                         uint8_t* __restrict__ out, int64_t rows,
                                                                         int cols, int ksteps, int64_t groups) {
    const WaveTask t(groups, ksteps);
    if (!t.ok) return;
    const int n = t.count(cols);
    if (n == 0) return;
    const uint32_t bytes = *reinterpret_cast<const uint32_t*>(scales + t.scale_at(ksteps));
    uint4 q[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) q[f] = *reinterpret_cast<const uint4*>(codes + t.code_at(f, ksteps));
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const int64_t row = t.row(f);
        if (row >= rows) continue;
        const uint32_t sb = (bytes >> (8 * f)) & 255u;
        const float s = sb == 255u ? bits_f32(0x7fc00000u) : mx_scale_f32(sb);
        const uint32_t w[4] = {q[f].x, q[f].y, q[f].z, q[f].w};
        float v[32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x2_t a = codes_to_f32<0>(w[i], s), b = codes_to_f32<1>(w[i], s);
            const f32x2_t c = codes_to_f32<2>(w[i], s), d = codes_to_f32<3>(w[i], s);
            v[8 * i] = a[0], v[8 * i + 1] = a[1], v[8 * i + 2] = b[0], v[8 * i + 3] = b[1];
            v[8 * i + 4] = c[0], v[8 * i + 5] = c[1], v[8 * i + 6] = d[0], v[8 * i + 7] = d[1];
        }
        uint8_t* o = out + (row * cols + static_cast<int64_t>(t.step) * kMxStepK + t.kb * kMxBlock) * kMxElemBytes<T>;
        if (n == kMxBlock) {
#pragma unroll
            for (int i = 0; i < MxRaw<T>::kVecs; ++i) {
                uint32_t r[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (T == kMxF32) r[j] = f32_bits(v[4 * i + j]);
                    else r[j] = f32x2_to_out_bits<T == kMxBf16>(v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
                }
                __builtin_memcpy(o + 16 * i, r, 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                if (i >= n) continue;
                if constexpr (T == kMxF32) reinterpret_cast<float*>(o)[i] = v[i];
                else reinterpret_cast<uint16_t*>(o)[i] = f32_to_out_bits<T == kMxBf16>(v[i]);
            }
        }
    }
}

// Row-major codes (rows, blocks * 16) and scales (rows, blocks) of a checkpoint
// -> packed (kBack: the other way). Blocks beyond the last become zeros.
template <bool kBack>
__global__ __launch_bounds__(64 * kWavesPerBlock) void repack_kernel(uint8_t* __restrict__ codes_rows,
                                                                     uint8_t* __restrict__ scales_rows,
                                                                     uint8_t* __restrict__ codes,
                                                                     uint8_t* __restrict__ scales, int64_t rows,
                                                                     int blocks, int ksteps, int64_t groups) {
    const WaveTask t(groups, ksteps);
    if (!t.ok) return;
    const int block = t.step * 4 + t.kb;
    uint32_t bytes = kBack ? *reinterpret_cast<const uint32_t*>(scales + t.scale_at(ksteps)) : 0u;
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const int64_t row = t.row(f);
        const bool have = row < rows && block < blocks;
        const int64_t at = row * blocks + block;
        uint4* packed = reinterpret_cast<uint4*>(codes + t.code_at(f, ksteps));
        if constexpr (kBack) {
            if (!have) continue;
            const uint4 q = *packed;
            __builtin_memcpy(codes_rows + at * 16, &q, 16);
            scales_rows[at] = static_cast<uint8_t>(bytes >> (8 * f));
        } else {
            uint4 q = make_uint4(0u, 0u, 0u, 0u);
            if (have) {
                q = load16_unaligned(codes_rows + at * 16);
                bytes |= static_cast<uint32_t>(scales_rows[at]) << (8 * f);
            }
            *packed = q;
        }
    }
    if constexpr (!kBack) *reinterpret_cast<uint32_t*>(scales + t.scale_at(ksteps)) = bytes;
}

struct Grid {
    int64_t groups;
    int ksteps;
    unsigned blocks;
    Grid(int64_t rows, int64_t cols)
        : groups(mx_groups(rows)), ksteps(static_cast<int>(mx_ksteps(cols))),
          blocks(static_cast<unsigned>((groups * ksteps + kWavesPerBlock - 1) / kWavesPerBlock)) {}
};

int launched() { return hipGetLastError() == hipSuccess ? FEATHER_OK : FEATHER_ERR_LAUNCH; }

}  // namespace

int mx_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, uint8_t* codes,
                uint8_t* scales, hipStream_t stream) {
    const Grid g(rows, cols);
    const uint8_t* xb = static_cast<const uint8_t*>(x);
    const int c = static_cast<int>(cols);
    if (dtype == kMxF16)
        quantize_kernel<kMxF16><<<g.blocks, 64 * kWavesPerBlock, 0, stream>>>(xb, rows, c, row_stride * 2, codes, scales, g.ksteps, g.groups);
    else if (dtype == kMxBf16)
        quantize_kernel<kMxBf16><<<g.blocks, 64 * kWavesPerBlock, 0, stream>>>(xb, rows, c, row_stride * 2, codes, scales, g.ksteps, g.groups);
    else
        quantize_kernel<kMxF32><<<g.blocks, 64 * kWavesPerBlock, 0, stream>>>(xb, rows, c, row_stride * 4, codes, scales, g.ksteps, g.groups);
    return launched();
}

int mx_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int dtype, int64_t rows, int64_t cols,
                  hipStream_t stream) {
    const Grid g(rows, cols);
    uint8_t* ob = static_cast<uint8_t*>(out);
    const int c = static_cast<int>(cols);
    if (dtype == kMxF16)
        dequantize_kernel<kMxF16><<<g.blocks, 64 * kWavesPerBlock, 0, stream>>>(codes, scales, ob, rows, c, g.ksteps, g.groups);
    else if (dtype == kMxBf16)
        dequantize_kernel<kMxBf16><<<g.blocks, 64 * kWavesPerBlock, 0, stream>>>(codes, scales, ob, rows, c, g.ksteps, g.groups);
    else
        dequantize_kernel<kMxF32><<<g.blocks, 64 * kWavesPerBlock, 0, stream>>>(codes, scales, ob, rows, c, g.ksteps, g.groups);
    return launched();
}

int mx_prepack(const uint8_t* codes_rows, const uint8_t* scales_rows, uint8_t* codes, uint8_t* scales, int64_t rows,
               int64_t cols, hipStream_t stream) {
    const Grid g(rows, cols);
    repack_kernel<false><<<g.blocks, 64 * kWavesPerBlock, 0, stream>>>(
        const_cast<uint8_t*>(codes_rows), const_cast<uint8_t*>(scales_rows), codes, scales, rows,
        static_cast<int>((cols + kMxBlock - 1) / kMxBlock), g.ksteps, g.groups);
    return launched();
}

int mx_unprepack(const uint8_t* codes, const uint8_t* scales, uint8_t* codes_rows, uint8_t* scales_rows, int64_t rows,
                 int64_t cols, hipStream_t stream) {
    const Grid g(rows, cols);
    repack_kernel<true><<<g.blocks, 64 * kWavesPerBlock, 0, stream>>>(
        codes_rows, scales_rows, const_cast<uint8_t*>(codes), const_cast<uint8_t*>(scales), rows,
        static_cast<int>((cols + kMxBlock - 1) / kMxBlock), g.ksteps, g.groups);
    return launched();
}

}  // namespace feather
