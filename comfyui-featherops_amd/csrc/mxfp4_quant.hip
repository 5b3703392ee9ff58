// MXFP4 quantisation and its layouts: row-major values <-> packed operands, and
// the row-major codes of checkpoints <-> packed operands. Formats in mxfp4.h.
//
// All four kernels give one wave rows of one step of 128 columns, a row tile of 16 or a
// group of four: lane l has row l % 16 of a tile and the block of 32 columns l / 16, the
// packed layout's own order, so a tile's codes are one KB. Values are read and written four
// lanes to a block (MxPieces). HBM bound: 13824 x 5120 in bf16 quantised at 5.6 TB/s (31.8 us),
// read back at 6.6 (27.1 us; the codes come from the memory-side cache).
#include <type_traits>

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
        return ((group * ksteps + step) * 4 + f) * 1024 + lane * 16;
    }
    __device__ __forceinline__ int64_t scale_at(int ksteps) const { return (group * ksteps + step) * 256 + lane * 4; }
    // the first column of the lane's pieces, and how many of their 8 values exist
    __device__ __forceinline__ int col() const { return step * kMxStepK + mx_piece_col(lane); }
    __device__ __forceinline__ int count(int cols) const { return max(0, min(8, cols - col())); }
};

// A wave quantises one row tile of one step: the other kernels' four tiles a wave leave too few waves to fill the
// chip below some thousand rows (154 x 4096 in bf16 2.5 against 3.3 us, 1003 x 3211 in fp16 3.8 against 6.7) and
// gain little above (13824 x 5120 31.8 against 31.2).
template <int T>
__global__ __launch_bounds__(64 * kWavesPerBlock) void quantize_kernel(const uint8_t* __restrict__ x, int64_t rows,
                                                                       int cols, int64_t row_bytes,
                                                                       uint8_t* __restrict__ codes,
                                                                       uint8_t* __restrict__ scales, int ksteps,
                                                                       int64_t tiles) {
    const int64_t w = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + (threadIdx.x >> 6);
    if (w >= tiles * ksteps) return;
    const int64_t tile = w / ksteps;
    const int step = static_cast<int>(w - tile * ksteps);
    const int lane = threadIdx.x & 63;
    const int col = step * kMxStepK + mx_piece_col(lane);
    // rows past the last repeat it: nothing reads what their place in the operand holds
    auto row = [&](int i) { return x + min(tile * 16 + mx_piece_row(lane, i), rows - 1) * row_bytes; };
    MxPieces<T> v;
    if ((step + 1) * kMxStepK <= cols) {  // (the same for the whole wave, as are the others)
#pragma unroll
        for (int i = 0; i < 4; ++i) v.load(i, row(i) + static_cast<int64_t>(col) * kMxElemBytes<T>);
    } else if (cols >= 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v.load_end(i, row(i), col, cols);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v.load_few(i, row(i) + static_cast<int64_t>(col) * kMxElemBytes<T>, cols - col);
    }
    uint32_t scale;
    const uint4 q = v.quantize(lane, &scale);
    const int64_t unit = (tile >> 2) * ksteps + step;
    *reinterpret_cast<uint4*>(codes + (unit * 4 + (tile & 3)) * 1024 + lane * 16) = q;
    scales[unit * 256 + lane * 4 + (tile & 3)] = static_cast<uint8_t>(scale);
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
    const uint32_t bytes = *reinterpret_cast<const uint32_t*>(scales + t.scale_at(ksteps));
    uint4 q[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) q[f] = *reinterpret_cast<const uint4*>(codes + t.code_at(f, ksteps));
    const int n = t.count(cols);
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const uint32_t sb = (bytes >> (8 * f)) & 255u;
        const uint32_t scale = sb == 255u ? 0x7fc00000u : f32_bits(mx_scale_f32(sb));
        const float by[4] = {bits_f32(quad_perm<kQuadLane[0]>(scale)), bits_f32(quad_perm<kQuadLane[1]>(scale)),
                             bits_f32(quad_perm<kQuadLane[2]>(scale)), bits_f32(quad_perm<kQuadLane[3]>(scale))};
        uint32_t w[4] = {q[f].x, q[f].y, q[f].z, q[f].w};
        quad_transpose(w, t.lane);  // piece i: 8 codes of the block of lane 4 (l / 4) + i
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = t.group * 64 + f * 16 + mx_piece_row(t.lane, i);
            if (row >= rows || n == 0) continue;
            const f32x2_t a = codes_to_f32<0>(w[i], by[i]), b = codes_to_f32<1>(w[i], by[i]);
            const f32x2_t c = codes_to_f32<2>(w[i], by[i]), d = codes_to_f32<3>(w[i], by[i]);
            const float v[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
            uint32_t r[MxPieces<T>::kVecs * 4];
#pragma unroll
            for (int k = 0; k < MxPieces<T>::kVecs * 4; ++k) {
                if constexpr (T == kMxF32) r[k] = f32_bits(v[k]);
                else r[k] = mx_round_pair<T == kMxBf16>(v[2 * k], v[2 * k + 1]);
            }
            uint8_t* o = out + (row * cols + t.col()) * kMxElemBytes<T>;
            if (n == 8) {
                __builtin_memcpy(o, r, sizeof(r));
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (k >= n) continue;
                    if constexpr (T == kMxF32) reinterpret_cast<uint32_t*>(o)[k] = r[k];
                    else reinterpret_cast<uint16_t*>(o)[k] = static_cast<uint16_t>(r[k >> 1] >> (16 * (k & 1)));
                }
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
    const int ksteps = static_cast<int>(mx_ksteps(cols));
    const int64_t tiles = (rows + 15) / 16;
    const unsigned blocks = static_cast<unsigned>((tiles * ksteps + kWavesPerBlock - 1) / kWavesPerBlock);
    auto go = [&](auto t) {
        quantize_kernel<t><<<blocks, 64 * kWavesPerBlock, 0, stream>>>(static_cast<const uint8_t*>(x), rows,
                                                                       static_cast<int>(cols), row_stride * kMxElemBytes<t>,
                                                                       codes, scales, ksteps, tiles);
    };
    if (dtype == kMxF16) go(std::integral_constant<int, kMxF16>{});
    else if (dtype == kMxBf16) go(std::integral_constant<int, kMxBf16>{});
    else go(std::integral_constant<int, kMxF32>{});
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
