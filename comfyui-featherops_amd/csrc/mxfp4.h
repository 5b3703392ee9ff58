// MXFP4: 32 consecutive values of a row share one power of two, each held in 4
// bits. The formats, their packed layout in HBM and the helpers that every
// kernel of this family uses.
//
//   code   e2m1 [s:1][e:2][m:1]: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives;
//          the earlier value of a pair in the low half of its byte
//   scale  e8m0: byte b stands for 2^(b - 127), 255 for NaN
//
// A block of 32 values with largest magnitude amax takes the scale
// 2^max(floor(log2 amax) - 2, -127) (so amax / scale is in [4, 8)) and the codes
// nearest to v / scale, ties to the even code, 6 beyond 6. A NaN or an infinity
// in the block makes it NaN as a whole (scale 255): a 4-bit code holds neither,
// and a block scaled by infinity would turn its other values to zero unseen.
//
// Packed layout, the operand order of the block-scaled 16x16x128 MFMA, for R
// rows and K columns, ksteps = ceil(K / 128), groups = ceil(R / 64):
//   codes  [groups][ksteps][4][64][16 bytes]: lane l of row tile f of group g and
//          step s holds row 64 g + 16 f + l % 16, columns 128 s + 32 (l / 16) .. + 31
//   scales [groups][ksteps][64][4]: byte f of lane l belongs to that row and block
// so a wave's operand load is one contiguous KB, the scales of four row tiles are one
// dword per lane, selected by the instruction, and the row tiles that a workgroup reads
// at one step are runs of 4 KB (with the steps of a row tile next to each other instead,
// M=333 N=K=5120 takes 12.7 us for 12.2). Columns beyond K are zero
// codes under scale 2^-127; rows beyond R may hold anything (no row's result
// depends on another row).
#pragma once

#include <type_traits>
#include <utility>

#include "feather_common.h"

namespace feather {

template <int... I, class F>
__device__ __forceinline__ void unrolled_impl(std::integer_sequence<int, I...>, F&& f) {
    (f(std::integral_constant<int, I>{}), ...);
}
// f(0_c) .. f(n-1_c): indices as constants, which the MFMA's scale selectors need.
template <int N, class F>
__device__ __forceinline__ void unrolled(F&& f) {
    unrolled_impl(std::make_integer_sequence<int, N>{}, f);
}

constexpr int kMxBlock = 32;
constexpr int kMxStepK = 128;
constexpr int kMxGroupRows = 64;

__host__ __device__ inline int64_t mx_ksteps(int64_t cols) { return (cols + kMxStepK - 1) / kMxStepK; }
__host__ __device__ inline int64_t mx_groups(int64_t rows) { return (rows + kMxGroupRows - 1) / kMxGroupRows; }

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// The scale byte of a block whose largest magnitude is amax (not negative; any
// NaN or infinity among the block's values arrives as one).
__device__ __forceinline__ uint32_t mx_scale_byte(float amax) {
    const uint32_t e = f32_bits(amax) >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// The scale as the fp32 operand of the conversion instructions (2^-127 is a
// subnormal, which they take; checked on gfx950 for every scale byte).
__device__ __forceinline__ float mx_scale_f32(uint32_t byte) {
    return bits_f32(byte == 0u ? 0x00400000u : byte << 23);
}

// The larger of |a| and |b| as bits: integer order is magnitude order, with
// infinities and NaN above every finite value.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a),
                                                                  __builtin_bit_cast(u16x2_t, b)));
}

// 16 bytes at any 2-byte alignment (global memory takes unaligned 16-byte
// accesses; an aligned one costs nothing extra).
__device__ __forceinline__ uint4 load16_unaligned(const void* p) {
    uint4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// Two fp32 -> fp16 or bf16 packed (a in the low half), round to nearest even: one instruction (a NaN keeps
// its payload, where f32x2_to_out_bits makes a bf16 one canonical with six more).
template <bool kBf16>
__device__ __forceinline__ uint32_t mx_round_pair(float a, float b) {
    if constexpr (kBf16) return f32x2_to_bf16x2_raw(a, b);
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, f16x2_t));
}

// The first n of 8 values from p, zeros beyond: kF32 ? 8 : 4 words.
template <bool kF32>
__device__ __forceinline__ void load_few8(const uint8_t* p, int n, uint32_t (&w)[kF32 ? 8 : 4]) {
#pragma unroll
    for (int k = 0; k < (kF32 ? 8 : 4); ++k) {
        if constexpr (kF32) {
            w[k] = k < n ? reinterpret_cast<const uint32_t*>(p)[k] : 0u;
        } else {
            const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
            w[k] = (2 * k < n ? static_cast<uint32_t>(q[2 * k]) : 0u) |
                   (2 * k + 1 < n ? static_cast<uint32_t>(q[2 * k + 1]) << 16 : 0u);
        }
    }
}

enum MxType { kMxF16 = 0, kMxBf16 = 1, kMxF32 = 2 };
template <int T>
constexpr int kMxElemBytes = T == kMxF32 ? 4 : 2;

template <int kCtrl>
__device__ __forceinline__ uint32_t quad_perm(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xf, 0xf, true));
}
constexpr int kQuadXor1 = 0xB1, kQuadXor2 = 0x4E;
constexpr int kQuadLane[4] = {0x00, 0x55, 0xAA, 0xFF};

// Transposes 4 x 4 dwords over four neighbouring lanes: lane s's r[v] becomes lane v's r[s].
__device__ __forceinline__ void quad_transpose(uint32_t (&r)[4], int lane) {
    const bool odd = lane & 1, high = lane & 2;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t got = quad_perm<kQuadXor1>(odd ? r[i] : r[i + 1]);
        if (odd) r[i] = got;
        else r[i + 1] = got;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t got = quad_perm<kQuadXor2>(high ? r[i] : r[i + 2]);
        if (high) r[i] = got;
        else r[i + 2] = got;
    }
}

// A wave's 16 rows x 128 columns of values on their way to (or from) an operand fragment, in which lane l
// has row l % 16 and block l / 16. In memory order four neighbouring lanes share the rows' 64-byte
// (16-bit values) runs instead: piece v of lane l is values 8 (l % 4) .. + 7 of the block that belongs to
// lane 4 (l / 4) + v, row 4 (l / 4) % 16 + v. A load then touches 64 contiguous bytes per four lanes
// where whole blocks per lane would touch 16 bytes of each of 64 runs; the codes, a quarter of the
// values' size, are transposed afterwards.
__device__ __forceinline__ int mx_piece_row(int lane, int v) { return (lane & 12) + v; }
__device__ __forceinline__ int mx_piece_col(int lane) { return (lane >> 4) * kMxBlock + (lane & 3) * 8; }

template <int T>
struct MxPieces {
    static constexpr int kVecs = T == kMxF32 ? 2 : 1;  // 16-byte vectors of a piece
    uint4 v[4][kVecs];

    // piece i from p
    __device__ __forceinline__ void load(int i, const uint8_t* p) {
#pragma unroll
        for (int k = 0; k < kVecs; ++k) v[i][k] = load16_unaligned(p + 16 * k);
    }
    // piece i, from column col on, of a row that ends within or before it and has cols >= 8 values: loaded
    // to end with the row and moved into place, zeros beyond
    __device__ __forceinline__ void load_end(int i, const uint8_t* row, int col, int cols) {
        const int from = min(col, cols - 8);
        load(i, row + from * kMxElemBytes<T>);
        const int by = col - from;
        if constexpr (T == kMxF32) {
            uint32_t w[8] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w, v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w};
#pragma unroll
            for (int s = 4; s >= 1; s /= 2)
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = by & s ? (k + s < 8 ? w[k + s] : 0u) : w[k];
            v[i][0] = make_uint4(w[0], w[1], w[2], w[3]);
            v[i][1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else {
            uint32_t w[4] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w};
#pragma unroll
            for (int s = 2; s >= 1; s /= 2)
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = by & (2 * s) ? (k + s < 4 ? w[k + s] : 0u) : w[k];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = by & 1 ? (w[k] >> 16) | (k < 3 ? w[k + 1] << 16 : 0u) : w[k];
            v[i][0] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (by >= 8) {
#pragma unroll
            for (int k = 0; k < kVecs; ++k) v[i][k] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    // the same for a row of fewer than 8 values: the n from p on
    __device__ __forceinline__ void load_few(int i, const uint8_t* p, int n) {
        uint32_t w[kVecs * 4];
        load_few8<T == kMxF32>(p, n, w);
#pragma unroll
        for (int k = 0; k < kVecs; ++k) v[i][k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    }

    // the codes of the lane's own block; *scale_byte gets its scale
    __device__ __forceinline__ uint4 quantize(int lane, uint32_t* scale_byte) const {
        uint32_t w[4][kVecs * 4], amax[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int k = 0; k < kVecs; ++k) {
                w[i][4 * k] = v[i][k].x;
                w[i][4 * k + 1] = v[i][k].y;
                w[i][4 * k + 2] = v[i][k].z;
                w[i][4 * k + 3] = v[i][k].w;
            }
            uint32_t m = 0u;
            if constexpr (T == kMxF32) {
#pragma unroll
                for (int k = 0; k < 8; ++k) m = max(m, w[i][k] & 0x7fffffffu);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) m = max_u16x2(m, w[i][k] & 0x7fff7fffu);
                m = max(m & 0xffffu, m >> 16);
            }
            m = max(m, quad_perm<kQuadXor1>(m));
            amax[i] = max(m, quad_perm<kQuadXor2>(m));
        }
        // every lane works out its own block's scale and hands it to the four that convert the block
        const int s = lane & 3;
        const uint32_t own = s & 2 ? (s & 1 ? amax[3] : amax[2]) : (s & 1 ? amax[1] : amax[0]);
        *scale_byte = mx_scale_byte(T == kMxF32    ? bits_f32(own)
                                    : T == kMxBf16 ? bits_f32(own << 16)
                                                   : half_bits_to_f32(static_cast<uint16_t>(own)));
        const uint32_t scale = f32_bits(mx_scale_f32(*scale_byte));
        const float by[4] = {bits_f32(quad_perm<kQuadLane[0]>(scale)), bits_f32(quad_perm<kQuadLane[1]>(scale)),
                             bits_f32(quad_perm<kQuadLane[2]>(scale)), bits_f32(quad_perm<kQuadLane[3]>(scale))};
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t c = 0u;
            if constexpr (T == kMxF32) {
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, bits_f32(w[i][0]), bits_f32(w[i][1]), by[i], 0);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, bits_f32(w[i][2]), bits_f32(w[i][3]), by[i], 1);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, bits_f32(w[i][4]), bits_f32(w[i][5]), by[i], 2);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, bits_f32(w[i][6]), bits_f32(w[i][7]), by[i], 3);
            } else if constexpr (T == kMxBf16) {
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[i][0]), by[i], 0);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[i][1]), by[i], 1);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[i][2]), by[i], 2);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[i][3]), by[i], 3);
            } else {
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, w[i][0]), by[i], 0);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, w[i][1]), by[i], 1);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, w[i][2]), by[i], 2);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(f16x2_t, w[i][3]), by[i], 3);
            }
            o[i] = c;
        }
        quad_transpose(o, lane);
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
};

// D(16x16, fp32) += A(16x128) * B(128x16), both MXFP4. Lane l supplies row
// (column) l % 16 and columns (rows) 32 (l / 16) .. + 31 as 16 bytes, and that
// block's scale in byte kByteA (kByteB) of its scale register; it receives D rows
// 4 (l / 16) .. + 3 of column l % 16. Checked against 64-bit sums on gfx950.
template <int kByteA, int kByteB>
__device__ __forceinline__ f32x4 mfma_mx(uint4 a, uint4 b, f32x4 c, uint32_t scale_a, uint32_t scale_b) {
    const i32x8 a8 = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w), 0, 0, 0, 0};
    const i32x8 b8 = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w), 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, kByteA, static_cast<int>(scale_a), kByteB,
                                                            static_cast<int>(scale_b));
}

// Host side launches (mxfp4_quant.hip, mxfp4_mm.hip, mxfp4_rows.hip); sizes are
// checked by the C entries.
int mx_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, uint8_t* codes,
                uint8_t* scales, hipStream_t stream);
int mx_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int dtype, int64_t rows, int64_t cols,
                  hipStream_t stream);
int mx_prepack(const uint8_t* codes_rows, const uint8_t* scales_rows, uint8_t* codes, uint8_t* scales, int64_t rows,
               int64_t cols, hipStream_t stream);
int mx_unprepack(const uint8_t* codes, const uint8_t* scales, uint8_t* codes_rows, uint8_t* scales_rows, int64_t rows,
                 int64_t cols, hipStream_t stream);

// Operands of a product C (M, N) = A (M, K) . B (N, K)^T + bias.
struct MxMmArgs {
    const uint8_t* a;         // packed codes (a_type kMxPacked) or row-major 16-bit values
    const uint8_t* a_scales;  // packed scales, unused for 16-bit activations
    int a_type;               // kMxF16, kMxBf16 or kMxPacked
    int64_t a_stride;         // elements between rows of 16-bit activations
    const uint8_t* b;
    const uint8_t* b_scales;
    const uint16_t* bias;  // output type, or null
    uint16_t* c;
    int64_t M;
    int N, K;
    int out_bf16;
    uint8_t* ws;  // arrival counters, then fp32 partial sums
    size_t ws_bytes;
};
constexpr int kMxPacked = 3;
constexpr size_t kMxCounterBytes = 65536;

// Few rows (mxfp4_rows.hip; 16-bit activations if their rows are within reach of 32-bit offsets), or
// LDS tiles (mxfp4_mm.hip): packed activations. Workspace bytes: 0 for none.
constexpr int64_t kMxFewRows = 32;
inline bool mx_rows_in_reach(int64_t M, int64_t stride) { return M <= 1 || (M - 1) * stride <= (int64_t(1) << 29); }
size_t mx_rows_workspace(int64_t M, int64_t N, int64_t K);
size_t mx_tiles_workspace(int64_t M, int64_t N, int64_t K);
int mx_mm_rows(const MxMmArgs& p, hipStream_t stream);
int mx_mm_tiles(const MxMmArgs& p, hipStream_t stream);
// What they launch with that workspace: feather_mxfp4_mm_plan.
void mx_rows_parts(int64_t M, int64_t N, int64_t K, int64_t* plan);
void mx_tiles_parts(int64_t M, int64_t N, int64_t K, int64_t* plan);

}  // namespace feather
