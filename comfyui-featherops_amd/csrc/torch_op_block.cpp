// torch ops of the MXFP4 operators and the block norms over the C ABI (no
// counterpart in the reference):
//   feather_ops::quantize_mxfp4, dequantize_mxfp4, prepack_mxfp4, unprepack_mxfp4
//   feather_ops::mxfp4_mm          16-bit activations, quantised in the call
//   feather_ops::mxfp4_mm_packed   activations that are packed MXFP4 already
//   feather_ops::modulated_norm(_mxfp4), gated_residual_norm(_mxfp4)
// Arguments are checked before anything is launched; launches go to torch's current
// stream of the first tensor's device. Views whose rows have one stride are read in
// place, others are made contiguous first.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cstdint>
#include <tuple>

#include "featherops_amd.h"
#include "torch_workspace.h"

namespace {

using OptTensor = std::optional<at::Tensor>;

hipStream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check_status(int st, const char* what) {
    TORCH_CHECK(st == FEATHER_OK, what, " failed: ", feather_status_string(st), " (status ", st, ")");
}

int value_code(at::ScalarType t, const char* what) {
    switch (t) {
        case at::kHalf: return FEATHER_DTYPE_F16;
        case at::kBFloat16: return FEATHER_DTYPE_BF16;
        case at::kFloat: return FEATHER_DTYPE_F32;
        default: TORCH_CHECK(false, what, " must be float16, bfloat16 or float32, got ", t);
    }
    return -1;
}

// at::empty on `like`'s device; on the GPU without another round through the dispatcher.
at::Tensor empty_on(const at::Tensor& like, at::IntArrayRef shape, at::ScalarType dtype) {
    if (!like.is_cuda()) return at::empty(shape, like.options().dtype(dtype));
    return at::Tensor(at::detail::empty_cuda(shape, dtype, like.device(), std::nullopt));
}

// t as rows of `cols` contiguous values with one stride between them: in place where its strides
// allow, otherwise a copy. (A contiguous tensor, the usual case, costs no view.)
struct Rows {
    at::Tensor t;  // keeps the values alive until the launch
    const void* p = nullptr;
    int64_t n = 0, stride = 0;
};

Rows as_rows(const at::Tensor& t) {
    const int64_t cols = t.size(-1);
    if (t.is_contiguous()) return {t, t.data_ptr(), cols ? t.numel() / cols : 0, cols};
    at::Tensor r = t.dim() == 2 ? t : t.reshape({cols ? t.numel() / cols : 0, cols});
    if ((cols > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < 0)) r = r.contiguous();
    return {r, r.data_ptr(), r.size(0), r.stride(0)};
}

// A packed operand is one uint8 tensor: its codes, then its scales (one allocation a call where two would
// cost a microsecond more).
struct Packed {
    at::Tensor data;
    int64_t codes_bytes = 0;
    uint8_t* codes() const { return static_cast<uint8_t*>(data.data_ptr()); }
    uint8_t* scales() const { return codes() + codes_bytes; }
};

template <class Int>
Int packed_units(const Int& rows, const Int& cols) {
    return (rows + 63) / 64 * ((cols + 127) / 128);
}

Packed empty_packed(int64_t rows, int64_t cols, const at::Tensor& like) {
    const int64_t units = packed_units(rows, cols);
    return {empty_on(like, {units * 4352}, at::kByte), units * 4096};
}

// What is checked of arguments in the CUDA and the Meta kernels alike (there sizes may be symbolic).
void check_packed_shape(const at::Tensor& data, const c10::SymInt& rows, const c10::SymInt& cols, const char* what) {
    const c10::SymInt bytes = packed_units(rows, cols) * 4352;
    TORCH_CHECK(data.scalar_type() == at::kByte && data.dim() == 1 && data.sym_size(0) == bytes, what, " must be packed for (",
                rows, ", ", cols, "): ", bytes, " contiguous uint8");
}

Packed check_packed(const at::Tensor& data, int64_t rows, int64_t cols, const char* what) {
    TORCH_CHECK(data.is_cuda(), what, " must be a CUDA tensor");
    check_packed_shape(data, rows, cols, what);
    const int64_t units = packed_units(rows, cols);
    TORCH_CHECK(data.is_contiguous(), what, " must be packed for (", rows, ", ", cols, "): ", units * 4352, " contiguous uint8");
    TORCH_CHECK(reinterpret_cast<uintptr_t>(data.data_ptr()) % 16 == 0, what, " data pointer must be 16-byte aligned");
    return {data, units * 4096};
}

template <class Int>
Int rows_of(c10::ArrayRef<Int> shape) {
    Int n = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) n = n * shape[i];
    return n;
}
// shape with its last dimension replaced
template <class Int>
c10::SmallVector<Int, at::kDimVectorStaticSize> with_last(c10::ArrayRef<Int> shape, const Int& n) {
    c10::SmallVector<Int, at::kDimVectorStaticSize> v(shape.begin(), shape.end());
    v.back() = n;
    return v;
}

// The type code of x's values.
int check_values(const at::Tensor& x) {
    TORCH_CHECK(x.dim() >= 1 && x.sym_size(-1) >= 1, "x must have at least one column");
    return value_code(x.scalar_type(), "x");
}

template <class Int>
int check_dequantize(c10::ArrayRef<Int> shape, at::ScalarType dtype) {
    TORCH_CHECK(!shape.empty() && shape.back() >= 1, "q must have at least one column");
    return value_code(dtype, "dtype");
}

void check_prepack(const at::Tensor& codes, const at::Tensor& scales, const c10::SymInt& cols) {
    TORCH_CHECK(codes.device() == scales.device(), "codes and scales must be on the same device");
    TORCH_CHECK(codes.element_size() == 1 && scales.element_size() == 1, "codes and scales must be 1-byte types");
    const c10::SymInt blocks = (cols + 31) / 32;
    TORCH_CHECK(cols >= 1 && codes.dim() == 2 && scales.dim() == 2 && codes.sym_size(0) == scales.sym_size(0) &&
                    codes.sym_size(1) == blocks * 16 && scales.sym_size(1) == blocks,
                "codes must be (rows, ", blocks * 16, ") and scales (rows, ", blocks, ") for ", cols, " columns");
}

void check_unprepack(const c10::SymInt& rows, const c10::SymInt& cols) {
    TORCH_CHECK(rows >= 0 && cols >= 1, "rows must not be negative, cols must be positive");
}

const uint8_t* bytes(const at::Tensor& t) { return static_cast<const uint8_t*>(t.data_ptr()); }

at::Tensor quantize_mxfp4(const at::Tensor& x) {
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int code = check_values(x);
    const c10::DeviceGuard guard(x.device());
    const Rows r = as_rows(x);
    const Packed q = empty_packed(r.n, x.size(-1), x);
    check_status(feather_mxfp4_quantize(r.p, code, r.n, x.size(-1), r.stride, q.codes(), q.scales(), stream_of(x)),
                 "quantize_mxfp4");
    return q.data;
}

at::Tensor dequantize_mxfp4(const at::Tensor& data, at::IntArrayRef shape, at::ScalarType dtype) {
    const int code = check_dequantize(shape, dtype);
    const int64_t rows = rows_of(shape), cols = shape.back();
    const Packed q = check_packed(data, rows, cols, "q");
    const c10::DeviceGuard guard(data.device());
    const at::Tensor out = empty_on(data, shape, dtype);
    check_status(feather_mxfp4_dequantize(q.codes(), q.scales(), out.data_ptr(), code, rows, cols, stream_of(data)),
                 "dequantize_mxfp4");
    return out;
}

at::Tensor prepack_mxfp4(const at::Tensor& codes, const at::Tensor& scales, int64_t cols) {
    TORCH_CHECK(codes.is_cuda() && scales.is_cuda(), "codes and scales must be CUDA tensors");
    check_prepack(codes, scales, cols);
    const c10::DeviceGuard guard(codes.device());
    const at::Tensor c = codes.contiguous(), s = scales.contiguous();
    const Packed q = empty_packed(c.size(0), cols, c);
    check_status(feather_mxfp4_prepack(bytes(c), bytes(s), q.codes(), q.scales(), c.size(0), cols, stream_of(c)),
                 "prepack_mxfp4");
    return q.data;
}

std::tuple<at::Tensor, at::Tensor> unprepack_mxfp4(const at::Tensor& data, int64_t rows, int64_t cols) {
    check_unprepack(rows, cols);
    const Packed q = check_packed(data, rows, cols, "q");
    const c10::DeviceGuard guard(data.device());
    const int64_t blocks = (cols + 31) / 32;
    const at::Tensor c = at::empty({rows, blocks * 16}, data.options()), s = at::empty({rows, blocks}, data.options());
    check_status(feather_mxfp4_unprepack(q.codes(), q.scales(), static_cast<uint8_t*>(c.data_ptr()),
                                         static_cast<uint8_t*>(s.data_ptr()), rows, cols, stream_of(data)),
                 "unprepack_mxfp4");
    return {c, s};
}

void check_mm_out(const at::Tensor& a, const at::Tensor& b, const OptTensor& bias, const c10::SymInt& N, at::ScalarType out_dtype) {
    TORCH_CHECK(b.device() == a.device(), "b must be on the same device as a");
    TORCH_CHECK(out_dtype == at::kHalf || out_dtype == at::kBFloat16, "out_dtype must be float16 or bfloat16");
    if (bias.has_value()) {
        TORCH_CHECK(bias->device() == a.device(), "bias must be on the same device as a");
        TORCH_CHECK(bias->scalar_type() == out_dtype, "bias must have the output's dtype");
        TORCH_CHECK(bias->dim() == 1 && bias->sym_size(0) == N && (N == 1 || bias->sym_stride(0) == 1),
                    "bias must be contiguous with N (", N, ") elements");
    }
}

at::ScalarType check_mm(const at::Tensor& a, const at::Tensor& b, const c10::SymInt& N, const c10::SymInt& K,
                        const OptTensor& bias, std::optional<at::ScalarType> dtype) {
    TORCH_CHECK(a.scalar_type() == at::kHalf || a.scalar_type() == at::kBFloat16, "a must be float16 or bfloat16");
    TORCH_CHECK(N >= 1 && K >= 1, "b must have at least one row and one column");
    TORCH_CHECK(a.dim() >= 1 && a.sym_size(-1) == K, "a must have b's ", K, " columns");
    const at::ScalarType out_dtype = dtype.value_or(a.scalar_type());
    check_mm_out(a, b, bias, N, out_dtype);
    return out_dtype;
}

template <class Int>
void check_mm_packed(const at::Tensor& a, c10::ArrayRef<Int> a_shape, const at::Tensor& b, const Int& N, const Int& K,
                     const OptTensor& bias, at::ScalarType out_dtype) {
    TORCH_CHECK(N >= 1 && K >= 1, "b must have at least one row and one column");
    TORCH_CHECK(!a_shape.empty() && a_shape.back() == K, "a must have b's ", K, " columns");
    check_mm_out(a, b, bias, N, out_dtype);
}

// C of the given shape (its leading dimensions are A's rows)
at::Tensor run_mm(const void* a, const uint8_t* a_scales, int a_dtype, int64_t a_stride, const Packed& b,
                  const OptTensor& bias, at::IntArrayRef shape, int64_t K, at::ScalarType out_dtype) {
    const hipStream_t stream = stream_of(b.data);
    const int64_t M = rows_of(shape), N = shape.back();
    const at::Tensor c = empty_on(b.data, shape, out_dtype);
    const size_t ws_bytes = feather_mxfp4_mm_workspace_size(M, N, K, a_dtype);
    at::Tensor ws;
    if (ws_bytes) ws = feather::workspace_for(b.data.device(), stream, ws_bytes);
    check_status(feather_mxfp4_mm(a, a_scales, a_dtype, a_stride, b.codes(), b.scales(),
                                  bias.has_value() ? static_cast<const uint16_t*>(bias->data_ptr()) : nullptr,
                                  static_cast<uint16_t*>(c.data_ptr()), M, N, K,
                                  out_dtype == at::kBFloat16 ? FEATHER_DTYPE_BF16 : FEATHER_DTYPE_F16,
                                  ws_bytes ? ws.data_ptr() : nullptr, ws_bytes ? static_cast<size_t>(ws.numel()) : 0, stream),
                 "mxfp4_mm");
    return c;
}

at::Tensor mxfp4_mm(const at::Tensor& a, const at::Tensor& b, int64_t N, int64_t K, const OptTensor& bias,
                    std::optional<at::ScalarType> dtype) {
    TORCH_CHECK(a.is_cuda(), "a must be a CUDA tensor");
    const at::ScalarType out_dtype = check_mm(a, b, N, K, bias, dtype);
    const Packed w = check_packed(b, N, K, "b");
    const c10::DeviceGuard guard(a.device());
    const Rows r = as_rows(a);
    const at::DimVector shape = with_last(a.sizes(), N);
    const int code = a.scalar_type() == at::kHalf ? FEATHER_DTYPE_F16 : FEATHER_DTYPE_BF16;
    if (feather_mxfp4_mm_takes_16bit(r.n, N, K, r.stride))
        return run_mm(r.p, nullptr, code, r.stride, w, bias, shape, K, out_dtype);
    const Packed q = empty_packed(r.n, K, a);
    check_status(feather_mxfp4_quantize(r.p, code, r.n, K, r.stride, q.codes(), q.scales(), stream_of(a)), "mxfp4_mm");
    return run_mm(q.codes(), q.scales(), FEATHER_DTYPE_MXFP4, 0, w, bias, shape, K, out_dtype);
}

at::Tensor mxfp4_mm_packed(const at::Tensor& a, at::IntArrayRef a_shape, const at::Tensor& b, int64_t N, int64_t K,
                           const OptTensor& bias, at::ScalarType out_dtype) {
    check_mm_packed(a, a_shape, b, N, K, bias, out_dtype);
    const Packed q = check_packed(a, rows_of(a_shape), K, "a");
    const Packed w = check_packed(b, N, K, "b");
    const c10::DeviceGuard guard(a.device());
    return run_mm(q.codes(), q.scales(), FEATHER_DTYPE_MXFP4, 0, w, bias, with_last(a_shape, N), K, out_dtype);
}

// ---- norms ----

// A vector or one vector per group of rows: t broadcast against x (..., cols). Rows of x that
// share a row of t are consecutive unless t repeats along a leading dimension alone, in which
// case it is written out.
struct RowVectors {
    Rows rows;
    const void* p = nullptr;
    int64_t group = 1, stride = 0;
};

void check_row_vectors(const at::Tensor& x, const at::Tensor& t, const char* what) {
    TORCH_CHECK(t.device() == x.device(), what, " must be on the same device as x");
    value_code(t.scalar_type(), what);
    const c10::SymIntArrayRef xs = x.sym_sizes(), ts = t.sym_sizes();
    TORCH_CHECK(!ts.empty() && ts.back() == xs.back() && ts.size() <= xs.size(), what, " must end in x's ", xs.back(),
                " columns and broadcast against x");
    for (size_t i = 1; i <= ts.size(); ++i)
        TORCH_CHECK(ts[ts.size() - i] == 1 || ts[ts.size() - i] == xs[xs.size() - i], what, " must broadcast against x");
}

// (checked)
RowVectors row_vectors(const at::Tensor& x, const at::Tensor& t, at::ScalarType dtype) {
    const int64_t skip = x.dim() - t.dim();
    int64_t group = 1, i = x.dim() - 2;
    for (; i >= 0 && (i < skip || t.size(i - skip) == 1); --i) group *= x.size(i);
    bool whole = true;  // every dimension before the shared ones is t's own
    for (int64_t j = i; j >= 0; --j) {
        const int64_t n = j < skip ? 1 : t.size(j - skip);
        whole = whole && n == x.size(j);
    }
    if (!whole) group = 1;
    RowVectors r;
    r.rows = t.scalar_type() == dtype ? as_rows(whole ? t : t.expand(x.sizes()))
                                      : as_rows((whole ? t : t.expand(x.sizes())).to(dtype));
    r.p = r.rows.p;
    r.group = group > 0 ? group : 1;
    r.stride = r.rows.n > 1 ? r.rows.stride : 0;
    return r;
}

void check_column_vector(const at::Tensor& x, const at::Tensor& t, const char* what) {
    TORCH_CHECK(t.device() == x.device(), what, " must be on the same device as x");
    value_code(t.scalar_type(), what);
    TORCH_CHECK(t.dim() == 1 && t.sym_size(0) == x.sym_size(-1), what, " must have x's ", x.sym_size(-1), " columns");
}

// (checked)
at::Tensor column_vector(const at::Tensor& t, at::ScalarType dtype) {
    const at::Tensor c = t.scalar_type() == dtype ? t : t.to(dtype);
    return c.size(0) > 1 && c.stride(0) != 1 ? c.contiguous() : c;
}

// The tensors of a norm, any of which but x may be missing.
struct NormIn {
    const at::Tensor& x;
    const at::Tensor* h;
    const OptTensor &gate, &post_weight, &weight, &bias, &scale, &shift;
};
const OptTensor kNone;

// The block's type, h's or y's.
at::ScalarType check_norm(const NormIn& in, std::optional<at::ScalarType> out_dtype) {
    const at::Tensor& x = in.x;
    const at::Tensor* h = in.h;
    TORCH_CHECK(x.dim() >= 1 && x.sym_size(-1) >= 1 && x.sym_size(-1) <= 16384, "x must have 1 to 16384 columns");
    const int x_code = value_code(x.scalar_type(), "x");
    if (h) {
        TORCH_CHECK(h->device() == x.device(), "h must be on the same device as x");
        TORCH_CHECK(h->sym_sizes() == x.sym_sizes(), "h must have x's shape");
        TORCH_CHECK(!out_dtype.has_value() || *out_dtype == h->scalar_type(), "out_dtype must be h's dtype");
    }
    const at::ScalarType block = h ? h->scalar_type() : out_dtype.value_or(x.scalar_type());
    const int y_code = value_code(block, h ? "h" : "out_dtype");
    TORCH_CHECK(x_code == FEATHER_DTYPE_F32 || x_code == y_code, "x must be float32 or of the block's dtype (", block, ")");
    if (in.gate.has_value()) check_row_vectors(x, *in.gate, "gate");
    if (in.scale.has_value()) check_row_vectors(x, *in.scale, "scale");
    if (in.shift.has_value()) check_row_vectors(x, *in.shift, "shift");
    if (in.post_weight.has_value()) check_column_vector(x, *in.post_weight, "post_weight");
    if (in.weight.has_value()) check_column_vector(x, *in.weight, "weight");
    if (in.bias.has_value()) check_column_vector(x, *in.bias, "bias");
    return block;
}

struct NormOut {
    at::Tensor stream, y;
    Packed q;
};

NormOut run_norm(const NormIn& in, bool layer, double eps, double residual_scale, std::optional<at::ScalarType> out_dtype,
                 bool codes) {
    const auto& [x, h, gate, post_weight, weight, bias, scale, shift] = in;
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const at::ScalarType block = check_norm(in, out_dtype);
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    const int x_code = value_code(x.scalar_type(), "x"), y_code = value_code(block, "h");
    // the vectors share one type: the block's if they all have it, otherwise fp32
    at::ScalarType mods = block;
    for (const OptTensor* t : {&gate, &post_weight, &weight, &bias, &scale, &shift})
        if (t->has_value() && (*t)->scalar_type() != block) mods = at::kFloat;

    const c10::DeviceGuard guard(x.device());
    const Rows xr = as_rows(x);
    const Rows hr = h ? as_rows(*h) : Rows{};
    at::Tensor pw, w, b;
    RowVectors g, sc, sh;
    if (gate.has_value()) g = row_vectors(x, *gate, mods);
    if (scale.has_value()) sc = row_vectors(x, *scale, mods);
    if (shift.has_value()) sh = row_vectors(x, *shift, mods);
    if (scale.has_value() && shift.has_value() && sc.group != sh.group) {  // one for the rows, one for groups: both by row
        sc = row_vectors(x, scale->expand(x.sizes()), mods);
        sh = row_vectors(x, shift->expand(x.sizes()), mods);
    }
    if (post_weight.has_value()) pw = column_vector(*post_weight, mods);
    if (weight.has_value()) w = column_vector(*weight, mods);
    if (bias.has_value()) b = column_vector(*bias, mods);

    NormOut out;
    if (h) out.stream = empty_on(x, x.sizes(), x.scalar_type());
    if (codes) out.q = empty_packed(rows, cols, x);
    else out.y = empty_on(x, x.sizes(), block);
    feather_block_norm_args a{};
    a.x = xr.p;
    a.h = hr.p;
    a.gate = g.p;
    a.post_weight = pw.defined() ? pw.data_ptr() : nullptr;
    a.weight = w.defined() ? w.data_ptr() : nullptr;
    a.bias = b.defined() ? b.data_ptr() : nullptr;
    a.scale = sc.p;
    a.shift = sh.p;
    a.x_out = out.stream.defined() ? out.stream.data_ptr() : nullptr;
    a.y = codes ? nullptr : out.y.data_ptr();
    a.codes = codes ? out.q.codes() : nullptr;
    a.scales = codes ? out.q.scales() : nullptr;
    a.rows = rows;
    a.cols = cols;
    a.x_row_stride = xr.stride;
    a.h_row_stride = hr.stride;
    a.gate_group = g.group;
    a.gate_row_stride = g.stride;
    a.mod_group = scale.has_value() ? sc.group : sh.group;
    a.scale_row_stride = sc.stride;
    a.shift_row_stride = sh.stride;
    a.x_dtype = x_code;
    a.y_dtype = y_code;
    a.mod_dtype = value_code(mods, "mods");
    a.norm = layer ? 1 : 0;
    a.eps = static_cast<float>(eps);
    a.residual_scale = static_cast<float>(residual_scale);
    check_status(feather_block_norm(&a, stream_of(x)), h ? "gated_residual_norm" : "modulated_norm");
    return out;
}

at::Tensor modulated_norm(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, const OptTensor& scale,
                          const OptTensor& shift, bool layer, double eps, std::optional<at::ScalarType> out_dtype) {
    return run_norm({x, nullptr, kNone, kNone, weight, bias, scale, shift}, layer, eps, 1.0, out_dtype, false).y;
}

at::Tensor modulated_norm_mxfp4(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias,
                                const OptTensor& scale, const OptTensor& shift, bool layer, double eps) {
    return run_norm({x, nullptr, kNone, kNone, weight, bias, scale, shift}, layer, eps, 1.0, {}, true).q.data;
}

std::tuple<at::Tensor, at::Tensor> gated_residual_norm(const at::Tensor& x, const at::Tensor& h, const OptTensor& gate,
                                                       const OptTensor& post_weight, const OptTensor& weight,
                                                       const OptTensor& bias, const OptTensor& scale,
                                                       const OptTensor& shift, bool layer, double eps,
                                                       double residual_scale, std::optional<at::ScalarType> out_dtype) {
    const NormOut o = run_norm({x, &h, gate, post_weight, weight, bias, scale, shift}, layer, eps, residual_scale, out_dtype, false);
    return {o.stream, o.y};
}

std::tuple<at::Tensor, at::Tensor> gated_residual_norm_mxfp4(const at::Tensor& x, const at::Tensor& h,
                                                             const OptTensor& gate, const OptTensor& post_weight,
                                                             const OptTensor& weight, const OptTensor& bias,
                                                             const OptTensor& scale, const OptTensor& shift, bool layer,
                                                             double eps, double residual_scale) {
    const NormOut o = run_norm({x, &h, gate, post_weight, weight, bias, scale, shift}, layer, eps, residual_scale, {}, true);
    return {o.stream, o.q.data};
}

// ---- fake tensors: the checks of the kernels above, and the results' shapes ----

at::Tensor values_meta(c10::SymIntArrayRef shape, const at::Tensor& like, at::ScalarType dtype) {
    return at::empty_symint(shape, like.options().dtype(dtype));
}
at::Tensor packed_meta(const c10::SymInt& rows, const c10::SymInt& cols, const at::Tensor& like) {
    return values_meta({packed_units(rows, cols) * 4352}, like, at::kByte);
}

at::Tensor quantize_mxfp4_meta(const at::Tensor& x) {
    check_values(x);
    return packed_meta(rows_of(x.sym_sizes()), x.sym_size(-1), x);
}
at::Tensor dequantize_mxfp4_meta(const at::Tensor& data, c10::SymIntArrayRef shape, at::ScalarType dtype) {
    check_dequantize(shape, dtype);
    check_packed_shape(data, rows_of(shape), shape.back(), "q");
    return values_meta(shape, data, dtype);
}
at::Tensor prepack_mxfp4_meta(const at::Tensor& codes, const at::Tensor& scales, c10::SymInt cols) {
    check_prepack(codes, scales, cols);
    return packed_meta(codes.sym_size(0), cols, codes);
}
std::tuple<at::Tensor, at::Tensor> unprepack_mxfp4_meta(const at::Tensor& data, c10::SymInt rows, c10::SymInt cols) {
    check_unprepack(rows, cols);
    check_packed_shape(data, rows, cols, "q");
    const c10::SymInt blocks = (cols + 31) / 32;
    return {values_meta({rows, blocks * 16}, data, at::kByte), values_meta({rows, blocks}, data, at::kByte)};
}
at::Tensor mxfp4_mm_meta(const at::Tensor& a, const at::Tensor& b, c10::SymInt N, c10::SymInt K, const OptTensor& bias,
                         std::optional<at::ScalarType> dtype) {
    const at::ScalarType out_dtype = check_mm(a, b, N, K, bias, dtype);
    check_packed_shape(b, N, K, "b");
    return values_meta(with_last(a.sym_sizes(), N), a, out_dtype);
}
at::Tensor mxfp4_mm_packed_meta(const at::Tensor& a, c10::SymIntArrayRef a_shape, const at::Tensor& b, c10::SymInt N,
                                c10::SymInt K, const OptTensor& bias, at::ScalarType out_dtype) {
    check_mm_packed(a, a_shape, b, N, K, bias, out_dtype);
    check_packed_shape(a, rows_of(a_shape), K, "a");
    check_packed_shape(b, N, K, "b");
    return values_meta(with_last(a_shape, N), a, out_dtype);
}
at::Tensor modulated_norm_meta(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias, const OptTensor& scale,
                               const OptTensor& shift, bool, double, std::optional<at::ScalarType> out_dtype) {
    return values_meta(x.sym_sizes(), x, check_norm({x, nullptr, kNone, kNone, weight, bias, scale, shift}, out_dtype));
}
at::Tensor modulated_norm_mxfp4_meta(const at::Tensor& x, const OptTensor& weight, const OptTensor& bias,
                                     const OptTensor& scale, const OptTensor& shift, bool, double) {
    check_norm({x, nullptr, kNone, kNone, weight, bias, scale, shift}, {});
    return quantize_mxfp4_meta(x);
}
std::tuple<at::Tensor, at::Tensor> gated_residual_norm_meta(const at::Tensor& x, const at::Tensor& h, const OptTensor& gate,
                                                            const OptTensor& post_weight, const OptTensor& weight,
                                                            const OptTensor& bias, const OptTensor& scale,
                                                            const OptTensor& shift, bool, double, double,
                                                            std::optional<at::ScalarType> out_dtype) {
    const at::ScalarType block = check_norm({x, &h, gate, post_weight, weight, bias, scale, shift}, out_dtype);
    return {values_meta(x.sym_sizes(), x, x.scalar_type()), values_meta(x.sym_sizes(), x, block)};
}
std::tuple<at::Tensor, at::Tensor> gated_residual_norm_mxfp4_meta(const at::Tensor& x, const at::Tensor& h,
                                                                  const OptTensor& gate, const OptTensor& post_weight,
                                                                  const OptTensor& weight, const OptTensor& bias,
                                                                  const OptTensor& scale, const OptTensor& shift, bool,
                                                                  double, double) {
    check_norm({x, &h, gate, post_weight, weight, bias, scale, shift}, {});
    return {values_meta(x.sym_sizes(), x, x.scalar_type()), quantize_mxfp4_meta(x)};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(feather_ops, m) {
    m.def("quantize_mxfp4(Tensor x) -> Tensor");
    m.def("dequantize_mxfp4(Tensor data, SymInt[] shape, ScalarType dtype) -> Tensor");
    m.def("prepack_mxfp4(Tensor codes, Tensor scales, SymInt cols) -> Tensor");
    m.def("unprepack_mxfp4(Tensor data, SymInt rows, SymInt cols) -> (Tensor, Tensor)");
    m.def("mxfp4_mm(Tensor a, Tensor b, SymInt N, SymInt K, Tensor? bias, ScalarType? out_dtype) -> Tensor");
    m.def("mxfp4_mm_packed(Tensor a, SymInt[] a_shape, Tensor b, SymInt N, SymInt K, Tensor? bias, ScalarType out_dtype) -> Tensor");
    m.def("modulated_norm(Tensor x, Tensor? weight, Tensor? bias, Tensor? scale, Tensor? shift, bool layer, float eps, "
          "ScalarType? out_dtype) -> Tensor");
    m.def("modulated_norm_mxfp4(Tensor x, Tensor? weight, Tensor? bias, Tensor? scale, Tensor? shift, bool layer, "
          "float eps) -> Tensor");
    m.def("gated_residual_norm(Tensor x, Tensor h, Tensor? gate, Tensor? post_weight, Tensor? weight, Tensor? bias, "
          "Tensor? scale, Tensor? shift, bool layer, float eps, float residual_scale, ScalarType? out_dtype) -> "
          "(Tensor, Tensor)");
    m.def("gated_residual_norm_mxfp4(Tensor x, Tensor h, Tensor? gate, Tensor? post_weight, Tensor? weight, "
          "Tensor? bias, Tensor? scale, Tensor? shift, bool layer, float eps, float residual_scale) -> "
          "(Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(feather_ops, CUDA, m) {
    m.impl("quantize_mxfp4", &quantize_mxfp4);
    m.impl("dequantize_mxfp4", &dequantize_mxfp4);
    m.impl("prepack_mxfp4", &prepack_mxfp4);
    m.impl("unprepack_mxfp4", &unprepack_mxfp4);
    m.impl("mxfp4_mm", &mxfp4_mm);
    m.impl("mxfp4_mm_packed", &mxfp4_mm_packed);
    m.impl("modulated_norm", &modulated_norm);
    m.impl("modulated_norm_mxfp4", &modulated_norm_mxfp4);
    m.impl("gated_residual_norm", &gated_residual_norm);
    m.impl("gated_residual_norm_mxfp4", &gated_residual_norm_mxfp4);
}

TORCH_LIBRARY_IMPL(feather_ops, Meta, m) {
    m.impl("quantize_mxfp4", &quantize_mxfp4_meta);
    m.impl("dequantize_mxfp4", &dequantize_mxfp4_meta);
    m.impl("prepack_mxfp4", &prepack_mxfp4_meta);
    m.impl("unprepack_mxfp4", &unprepack_mxfp4_meta);
    m.impl("mxfp4_mm", &mxfp4_mm_meta);
    m.impl("mxfp4_mm_packed", &mxfp4_mm_packed_meta);
    m.impl("modulated_norm", &modulated_norm_meta);
    m.impl("modulated_norm_mxfp4", &modulated_norm_mxfp4_meta);
    m.impl("gated_residual_norm", &gated_residual_norm_meta);
    m.impl("gated_residual_norm_mxfp4", &gated_residual_norm_mxfp4_meta);
}
