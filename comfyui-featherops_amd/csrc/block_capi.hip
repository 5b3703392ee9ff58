// extern "C" entry points of the MXFP4 operators and the block norms (declared in
// include/featherops_amd.h). Sizes, types and pointers are checked here, before
// anything is launched.
#include <initializer_list>

#include "block_norm.h"
#include "featherops_amd.h"
#include "mxfp4.h"

namespace {

using namespace feather;

constexpr int64_t kMaxCols = int64_t(1) << 24;
constexpr int64_t kMaxRows = int64_t(1) << 30;

// rows and cols of an MXFP4 tensor; the layout kernels give one wave at least 16 x 128 values and a
// grid holds fewer than 2^32 threads
bool mx_sizes_ok(int64_t rows, int64_t cols) {
    return rows >= 0 && cols > 0 && rows <= kMaxRows && cols < kMaxCols && mx_groups(rows) * mx_ksteps(cols) < (int64_t(1) << 23);
}
bool value_type(int t) { return t == FEATHER_DTYPE_F16 || t == FEATHER_DTYPE_BF16 || t == FEATHER_DTYPE_F32; }
// Packed buffers are read in 16-byte units, by copies into LDS among others.
bool aligned(std::initializer_list<const void*> packed) {
    uintptr_t bits = 0;
    for (const void* p : packed) bits |= reinterpret_cast<uintptr_t>(p);
    return bits % 16 == 0;
}
bool mm_sizes_ok(int64_t M, int64_t N, int64_t K) { return mx_sizes_ok(M, K) && N > 0 && mx_sizes_ok(N, K); }

}  // namespace

extern "C" {

size_t feather_mxfp4_codes_bytes(int64_t rows, int64_t cols) {
    return mx_sizes_ok(rows, cols) ? static_cast<size_t>(mx_groups(rows) * mx_ksteps(cols)) * 4096 : 0;
}

size_t feather_mxfp4_scales_bytes(int64_t rows, int64_t cols) {
    return mx_sizes_ok(rows, cols) ? static_cast<size_t>(mx_groups(rows) * mx_ksteps(cols)) * 256 : 0;
}

int feather_mxfp4_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t row_stride, uint8_t* codes,
                           uint8_t* scales, hipStream_t stream) {
    if (!mx_sizes_ok(rows, cols) || !value_type(x_dtype) || (rows > 1 && row_stride < 0)) return FEATHER_ERR_INVALID;
    if (rows == 0) return FEATHER_OK;
    if (!x || !codes || !scales || !aligned({codes, scales})) return FEATHER_ERR_INVALID;
    return mx_quantize(x, x_dtype, rows, cols, row_stride, codes, scales, stream);
}

int feather_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int out_dtype, int64_t rows,
                             int64_t cols, hipStream_t stream) {
    if (!mx_sizes_ok(rows, cols) || !value_type(out_dtype)) return FEATHER_ERR_INVALID;
    if (rows == 0) return FEATHER_OK;
    if (!codes || !scales || !out || !aligned({codes, scales})) return FEATHER_ERR_INVALID;
    return mx_dequantize(codes, scales, out, out_dtype, rows, cols, stream);
}

int feather_mxfp4_prepack(const uint8_t* codes_rows, const uint8_t* scales_rows, uint8_t* codes, uint8_t* scales,
                          int64_t rows, int64_t cols, hipStream_t stream) {
    if (!mx_sizes_ok(rows, cols)) return FEATHER_ERR_INVALID;
    if (rows == 0) return FEATHER_OK;
    if (!codes_rows || !scales_rows || !codes || !scales || !aligned({codes, scales})) return FEATHER_ERR_INVALID;
    return mx_prepack(codes_rows, scales_rows, codes, scales, rows, cols, stream);
}

int feather_mxfp4_unprepack(const uint8_t* codes, const uint8_t* scales, uint8_t* codes_rows, uint8_t* scales_rows,
                            int64_t rows, int64_t cols, hipStream_t stream) {
    if (!mx_sizes_ok(rows, cols)) return FEATHER_ERR_INVALID;
    if (rows == 0) return FEATHER_OK;
    if (!codes_rows || !scales_rows || !codes || !scales || !aligned({codes, scales})) return FEATHER_ERR_INVALID;
    return mx_unprepack(codes, scales, codes_rows, scales_rows, rows, cols, stream);
}

int feather_mxfp4_mm_takes_16bit(int64_t M, int64_t N, int64_t K, int64_t a_row_stride) {
    return mm_sizes_ok(M, N, K) && M <= kMxFewRows && mx_rows_in_reach(M, a_row_stride) ? 1 : 0;
}

size_t feather_mxfp4_mm_workspace_size(int64_t M, int64_t N, int64_t K, int a_dtype) {
    if (!mm_sizes_ok(M, N, K) || M == 0) return 0;
    return M <= kMxFewRows ? mx_rows_workspace(M, N, K) : mx_tiles_workspace(M, N, K);
}

int feather_mxfp4_mm_plan(int64_t M, int64_t N, int64_t K, int64_t* plan) {
    if (!mm_sizes_ok(M, N, K) || !plan) return FEATHER_ERR_INVALID;
    for (int i = 0; i < 8; ++i) plan[i] = 0;
    if (M == 0) return FEATHER_OK;
    if (M <= kMxFewRows) mx_rows_parts(M, N, K, plan);
    else mx_tiles_parts(M, N, K, plan);
    return FEATHER_OK;
}

int feather_mxfp4_mm(const void* a, const uint8_t* a_scales, int a_dtype, int64_t a_row_stride, const uint8_t* b,
                     const uint8_t* b_scales, const uint16_t* bias, uint16_t* c, int64_t M, int64_t N, int64_t K,
                     int output_dtype, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const bool packed = a_dtype == FEATHER_DTYPE_MXFP4;
    if (!mm_sizes_ok(M, N, K) || (!packed && a_dtype != FEATHER_DTYPE_F16 && a_dtype != FEATHER_DTYPE_BF16) ||
        (output_dtype != FEATHER_DTYPE_F16 && output_dtype != FEATHER_DTYPE_BF16))
        return FEATHER_ERR_INVALID;
    if (M == 0) return FEATHER_OK;
    if (!a || (packed && !a_scales) || !b || !b_scales || !c || (!packed && M > 1 && a_row_stride < 0))
        return FEATHER_ERR_INVALID;
    if (!aligned({b, b_scales}) || (packed && !aligned({a, a_scales}))) return FEATHER_ERR_INVALID;
    const MxMmArgs args{static_cast<const uint8_t*>(a), a_scales, a_dtype, a_row_stride, b, b_scales, bias, c, M,
                        static_cast<int>(N), static_cast<int>(K), output_dtype == FEATHER_DTYPE_BF16,
                        static_cast<uint8_t*>(workspace), workspace ? workspace_bytes : 0};
    if (M <= kMxFewRows) return mx_mm_rows(args, stream);
    if (!packed) return FEATHER_ERR_UNSUPPORTED;
    return mx_mm_tiles(args, stream);
}

int feather_block_norm(const feather_block_norm_args* p, hipStream_t stream) {
    if (!p || p->rows < 0 || p->rows > kMaxRows || p->cols <= 0 || p->cols > kNormMaxCols || !value_type(p->x_dtype) ||
        !value_type(p->y_dtype) || (p->x_dtype != FEATHER_DTYPE_F32 && p->x_dtype != p->y_dtype) ||
        (p->mod_dtype != FEATHER_DTYPE_F32 && p->mod_dtype != p->y_dtype) || (p->norm != 0 && p->norm != 1))
        return FEATHER_ERR_INVALID;
    if (p->rows == 0) return FEATHER_OK;
    const bool to_codes = p->codes || p->scales;
    if (!p->x || (p->h && !p->x_out) || (!p->h && (p->gate || p->post_weight)) || (p->gate && p->gate_group <= 0) ||
        ((p->scale || p->shift) && p->mod_group <= 0) || (to_codes ? !p->codes || !p->scales || p->y || !aligned({p->codes, p->scales}) : !p->y))
        return FEATHER_ERR_INVALID;
    auto group = [&](int64_t g) { return static_cast<uint32_t>(g < p->rows ? g : p->rows); };
    const NormArgs a{p->x, p->x_row_stride, p->h, p->h_row_stride, p->gate, p->gate_row_stride, p->scale,
                     p->scale_row_stride, p->shift, p->shift_row_stride, p->post_weight, p->weight, p->bias, p->x_out,
                     p->y, p->codes, p->scales, group(p->gate_group), group(p->mod_group), p->rows,
                     static_cast<int>(p->cols), p->x_dtype, p->y_dtype, p->mod_dtype == FEATHER_DTYPE_F32, p->norm,
                     p->eps, p->residual_scale, 0};
    return block_norm(a, stream);
}

}  // extern "C"
