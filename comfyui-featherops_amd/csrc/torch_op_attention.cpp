// torch ops of rotary positions and attention over the C ABI (no counterpart in the
// reference):
//   feather_ops::rope_table
//   feather_ops::norm_rope, qk_norm_rope
//   feather_ops::attention, packed_attention
// Arguments are checked before anything is launched; launches go to torch's current
// stream of the first tensor's device. Tensors whose last dimension is contiguous are read in
// place, others are made contiguous first.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cmath>
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

at::Tensor empty_on(const at::Tensor& like, at::IntArrayRef shape, at::ScalarType dtype) {
    return at::Tensor(at::detail::empty_cuda(shape, dtype, like.device(), std::nullopt));
}

void check_device(const at::Tensor& t, const at::Tensor& like, const char* what, const char* of) {
    TORCH_CHECK(t.device() == like.device(), what, " must be on the same device as ", of);
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

// ---- rotary positions ----

constexpr int64_t kMaxAxes = 8, kMaxDim = 256;

// The pairs that the axes have together.
int64_t check_table(const at::Tensor& positions, at::IntArrayRef axes, double theta) {
    TORCH_CHECK(!axes.empty() && static_cast<int64_t>(axes.size()) <= kMaxAxes, "there must be 1 to 8 axes");
    int64_t dims = 0;
    for (const int64_t d : axes) {
        TORCH_CHECK(d >= 0 && d % 2 == 0 && d <= kMaxDim, "an axis must have an even number of values, up to 256, got ", d);
        dims += d;
    }
    TORCH_CHECK(dims >= 2 && dims <= kMaxDim, "the axes must have 2 to 256 values together, got ", dims);
    TORCH_CHECK(theta > 0.0 && std::isfinite(theta), "theta must be positive and finite");
    TORCH_CHECK(positions.dim() >= 1 && positions.sym_size(-1) == static_cast<int64_t>(axes.size()), "positions must end in ",
                axes.size(), " axes");
    const at::ScalarType t = positions.scalar_type();
    TORCH_CHECK(t == at::kInt || t == at::kLong || t == at::kFloat || t == at::kDouble,
                "positions must be int32, int64, float32 or float64, got ", t);
    return dims / 2;
}

at::Tensor rope_table(const at::Tensor& positions, at::IntArrayRef axes, double theta, bool shared) {
    TORCH_CHECK(positions.is_cuda(), "positions must be a CUDA tensor");
    const int64_t pairs = check_table(positions, axes, theta);
    const c10::DeviceGuard guard(positions.device());
    const at::Tensor p = positions.contiguous();
    const int64_t rows = p.numel() / static_cast<int64_t>(axes.size());
    at::DimVector shape(p.sizes().begin(), p.sizes().end());
    shape.back() = pairs;
    shape.push_back(2);
    const at::Tensor table = empty_on(p, shape, at::kFloat);
    int dims[kMaxAxes], code = FEATHER_POSITION_F64;
    for (size_t i = 0; i < axes.size(); ++i) dims[i] = static_cast<int>(axes[i]);
    switch (p.scalar_type()) {
        case at::kInt: code = FEATHER_POSITION_I32; break;
        case at::kLong: code = FEATHER_POSITION_I64; break;
        case at::kFloat: code = FEATHER_POSITION_F32; break;
        default: break;
    }
    check_status(feather_rope_table(p.data_ptr(), code, rows, dims, static_cast<int>(axes.size()), theta, shared,
                                    static_cast<float*>(table.data_ptr()), stream_of(p)),
                 "rope_table");
    return table;
}

enum Norm { kNone = 0, kHead = 1, kRow = 2 };

void check_rope_side(const at::Tensor& x, const OptTensor& weight, int64_t norm, const char* what) {
    TORCH_CHECK(x.dim() == 3 || x.dim() == 4, what, " must be (tokens, heads, head_dim) or (batch, tokens, heads, head_dim)");
    const c10::SymInt dim = x.sym_size(-1), heads = x.sym_size(-2);
    TORCH_CHECK(heads >= 1 && heads <= 65536, what, " must have 1 to 65536 heads");
    TORCH_CHECK(dim >= 8 && dim <= kMaxDim && dim % 8 == 0, what, "'s head_dim must be a multiple of 8, up to 256, got ", dim);
    if (norm == kRow) {
        int64_t wide = 8;
        while (dim > wide) wide *= 2;
        TORCH_CHECK(heads * wide <= 16384, "a norm over the row takes up to 16384 values (head_dim rounded up to a power of two)");
    }
    if (weight.has_value()) {
        TORCH_CHECK(norm != kNone, "a weight needs a norm");
        check_device(*weight, x, "a weight", what);
        value_code(weight->scalar_type(), "a weight");
        const c10::SymInt n = norm == kRow ? heads * dim : dim;
        TORCH_CHECK(weight->dim() == 1 && weight->sym_size(0) == n, what, "'s weight must have ", n, " elements");
    }
}

void check_rope(const at::Tensor& q, const at::Tensor* k, const OptTensor& table, const OptTensor& q_weight,
                const OptTensor& k_weight, int64_t norm) {
    TORCH_CHECK(norm >= kNone && norm <= kRow, "norm must be 0, 1 or 2");
    value_code(q.scalar_type(), k ? "q" : "x");
    check_rope_side(q, q_weight, norm, k ? "q" : "x");
    if (k) {
        check_device(*k, q, "k", "q");
        TORCH_CHECK(k->scalar_type() == q.scalar_type(), "k must have q's dtype");
        TORCH_CHECK(k->dim() == q.dim() && k->sym_size(-1) == q.sym_size(-1) && k->sym_size(-3) == q.sym_size(-3) &&
                        k->sym_size(0) == q.sym_size(0),
                    "k must have q's batch, tokens and head_dim");
        check_rope_side(*k, k_weight, norm, "k");
    }
    if (table.has_value()) {
        check_device(*table, q, "table", k ? "q" : "x");
        TORCH_CHECK(table->scalar_type() == at::kFloat, "table must be float32");
        TORCH_CHECK((table->dim() == 3 || (table->dim() == 4 && q.dim() == 4)) && table->sym_size(-1) == 2 &&
                        table->sym_size(-2) >= 1 && table->sym_size(-2) * 2 <= q.sym_size(-1) &&
                        table->sym_size(-3) == q.sym_size(-3) && (table->dim() == 3 || table->sym_size(0) == q.sym_size(0) || table->sym_size(0) == 1),
                    "table must be (tokens, pairs, 2), or that for each sample, with at most head_dim / 2 pairs");
    }
}

// x with a contiguous last dimension, in place where it has one.
at::Tensor with_rows(const at::Tensor& x) { return x.size(-1) > 1 && x.stride(-1) != 1 ? x.contiguous() : x; }

std::tuple<at::Tensor, at::Tensor> run_rope(const at::Tensor& q, const at::Tensor* k, const OptTensor& table,
                                            const OptTensor& q_weight, const OptTensor& k_weight, int64_t norm, double eps,
                                            bool halves) {
    TORCH_CHECK(q.is_cuda(), k ? "q" : "x", " must be a CUDA tensor");
    check_rope(q, k, table, q_weight, k_weight, norm);
    const c10::DeviceGuard guard(q.device());
    const at::Tensor qr = with_rows(q), kr = k ? with_rows(*k) : at::Tensor();
    const at::ScalarType dtype = q.scalar_type();
    at::ScalarType weights = dtype;  // both weights have one type: the tensors', or else fp32
    for (const OptTensor* w : {&q_weight, &k_weight})
        if (w->has_value() && (*w)->scalar_type() != dtype) weights = at::kFloat;
    auto weight_of = [&](const OptTensor& w) {
        if (!w.has_value()) return at::Tensor();
        return (w->scalar_type() == weights ? *w : w->to(weights)).contiguous();
    };
    const at::Tensor qw = weight_of(q_weight), kw = weight_of(k_weight);
    at::Tensor t;
    if (table.has_value()) t = table->contiguous();
    const at::Tensor q_out = empty_on(q, q.sizes(), dtype), k_out = k ? empty_on(q, k->sizes(), dtype) : at::Tensor();

    feather_rope_args a{};
    const bool samples = q.dim() == 4;
    a.batch = samples ? q.size(0) : 1;
    a.tokens = q.size(-3);
    a.q = qr.data_ptr();
    a.q_out = q_out.data_ptr();
    a.q_weight = qw.defined() ? qw.data_ptr() : nullptr;
    a.q_heads = q.size(-2);
    a.q_batch_stride = samples ? qr.stride(0) : 0;
    a.q_token_stride = qr.stride(-3);
    a.q_head_stride = qr.stride(-2);
    if (k) {
        a.k = kr.data_ptr();
        a.k_out = k_out.data_ptr();
        a.k_weight = kw.defined() ? kw.data_ptr() : nullptr;
        a.k_heads = k->size(-2);
        a.k_batch_stride = samples ? kr.stride(0) : 0;
        a.k_token_stride = kr.stride(-3);
        a.k_head_stride = kr.stride(-2);
    }
    a.head_dim = q.size(-1);
    if (t.defined() && t.numel()) {
        a.table = static_cast<const float*>(t.data_ptr());
        a.pairs = t.size(-2);
        a.table_batch_stride = t.dim() == 4 && t.size(0) > 1 ? t.stride(0) : 0;
    }
    a.dtype = value_code(dtype, "q");
    a.weight_dtype = value_code(weights, "weights");
    a.norm = static_cast<int>(norm);
    a.pairs_of_halves = halves;
    a.eps = static_cast<float>(eps);
    check_status(feather_qk_norm_rope(&a, stream_of(q)), k ? "qk_norm_rope" : "norm_rope");
    return {q_out, k_out};
}

at::Tensor norm_rope(const at::Tensor& x, const OptTensor& table, const OptTensor& weight, int64_t norm, double eps, bool halves) {
    return std::get<0>(run_rope(x, nullptr, table, weight, {}, norm, eps, halves));
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& q, const at::Tensor& k, const OptTensor& table,
                                                const OptTensor& q_weight, const OptTensor& k_weight, int64_t norm, double eps,
                                                bool halves) {
    return run_rope(q, &k, table, q_weight, k_weight, norm, eps, halves);
}

// ---- attention ----

void check_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t dims, const char* shape) {
    TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16, "q must be float16 or bfloat16, got ",
                q.scalar_type());
    check_device(k, q, "k", "q");
    check_device(v, q, "v", "q");
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "k and v must have q's dtype");
    TORCH_CHECK(q.dim() == dims && k.dim() == dims && v.dim() == dims, "q, k and v must be ", shape);
    const c10::SymInt dim = q.sym_size(-1), heads = q.sym_size(-2), shared = k.sym_size(-2);
    TORCH_CHECK(dim >= 8 && dim <= kMaxDim && dim % 8 == 0, "head_dim must be a multiple of 8, up to 256, got ", dim);
    TORCH_CHECK(k.sym_size(-1) == dim && v.sym_sizes() == k.sym_sizes(), "k and v must have one shape, and q's head_dim");
    TORCH_CHECK(heads >= 1 && heads <= 65536 && shared >= 1 && heads % shared == 0, "q's heads (", heads,
                ") must be a multiple of k's (", shared, ")");
    const int64_t most = int64_t(1) << 30;
    TORCH_CHECK(q.sym_size(-3) <= most && k.sym_size(-3) <= most && q.sym_size(-3) * (heads / shared) <= most,
                "q and k may have up to 2^30 tokens, q's times the heads that share a key head too");
}

double check_scale(const at::Tensor& q, std::optional<double> scale) {
    if (scale.has_value()) {
        const float s = static_cast<float>(*scale);
        TORCH_CHECK(s > 0.0f && s <= 0x1p127f, "scale must be positive and at most 2^127");
        return *scale;
    }
    return 0.0;
}

void check_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptTensor& k_lengths, const OptTensor& mask) {
    check_qkv(q, k, v, 4, "(batch, tokens, heads, head_dim)");
    TORCH_CHECK(k.sym_size(0) == q.sym_size(0), "k must have q's batch");
    TORCH_CHECK(q.sym_size(0) <= 65536, "there may be up to 65536 samples");
    if (k_lengths.has_value()) {
        check_device(*k_lengths, q, "k_lengths", "q");
        TORCH_CHECK(k_lengths->scalar_type() == at::kInt && k_lengths->dim() == 1 && k_lengths->sym_size(0) == q.sym_size(0),
                    "k_lengths must be int32, one for each sample");
    }
    if (mask.has_value()) {
        check_device(*mask, q, "mask", "q");
        const at::ScalarType t = mask->scalar_type();
        TORCH_CHECK(t == at::kBool || t == at::kFloat || t == q.scalar_type(), "mask must be bool, float32 or of q's dtype, got ", t);
        TORCH_CHECK(mask->dim() >= 1 && mask->dim() <= 4, "mask must broadcast to (batch, heads, q tokens, k tokens)");
        const c10::SymInt full[4] = {q.sym_size(0), q.sym_size(2), q.sym_size(1), k.sym_size(1)};
        for (int64_t i = 0; i < mask->dim(); ++i)
            TORCH_CHECK(mask->sym_size(mask->dim() - 1 - i) == 1 || mask->sym_size(mask->dim() - 1 - i) == full[3 - i],
                        "mask must broadcast to (batch, heads, q tokens, k tokens)");
    }
}

void check_offsets(const at::Tensor& offsets, const at::Tensor& q, const char* what) {
    check_device(offsets, q, what, "q");
    TORCH_CHECK(offsets.scalar_type() == at::kInt && offsets.dim() == 1 && offsets.sym_size(0) >= 2 && offsets.sym_size(0) <= 65537, what,
                " must be int32, one more than there are sequences (1 to 65536)");
}

void check_packed_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& q_offsets,
                            const OptTensor& k_offsets) {
    check_qkv(q, k, v, 3, "(tokens, heads, head_dim)");
    check_offsets(q_offsets, q, "q_offsets");
    if (k_offsets.has_value()) {
        check_offsets(*k_offsets, q, "k_offsets");
        TORCH_CHECK(k_offsets->sym_size(0) == q_offsets.sym_size(0), "k_offsets must have q_offsets' size");
    } else {
        TORCH_CHECK(k.sym_size(0) == q.sym_size(0), "k must have q's tokens where there are no k_offsets");
    }
}

// x as the kernels read it: in place where its rows are contiguous and lie on 16-byte boundaries. Strides of
// dimensions of size 1 say nothing.
struct Operand {
    at::Tensor t;
    int64_t batch = 0, token = 0, head = 0;
};

Operand operand(const at::Tensor& x) {
    Operand o;
    auto take = [&](const at::Tensor& t) {
        o.t = t;
        o.batch = t.dim() == 4 && t.size(0) > 1 ? t.stride(0) : 0;
        o.token = t.size(-3) > 1 ? t.stride(-3) : 0;
        o.head = t.size(-2) > 1 ? t.stride(-2) : 0;
        return t.stride(-1) == 1 && (o.batch | o.token | o.head) % 8 == 0 && o.token < (int64_t(1) << 23) &&
               reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    };
    if (!take(x)) take(x.clone(at::MemoryFormat::Contiguous));
    return o;
}

at::Tensor run_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, feather_attention_args& a, bool causal,
                         std::optional<double> scale, const char* what) {
    const Operand qo = operand(q), ko = operand(k), vo = operand(v);
    const at::Tensor out = empty_on(q, q.sizes(), q.scalar_type());
    a.q = qo.t.data_ptr();
    a.k = ko.t.data_ptr();
    a.v = vo.t.data_ptr();
    a.out = out.data_ptr();
    a.q_tokens = q.size(-3);
    a.k_tokens = k.size(-3);
    a.heads = q.size(-2);
    a.kv_heads = k.size(-2);
    a.head_dim = q.size(-1);
    a.q_batch_stride = qo.batch, a.q_token_stride = qo.token, a.q_head_stride = qo.head;
    a.k_batch_stride = ko.batch, a.k_token_stride = ko.token, a.k_head_stride = ko.head;
    a.v_batch_stride = vo.batch, a.v_token_stride = vo.token, a.v_head_stride = vo.head;
    a.dtype = q.scalar_type() == at::kHalf ? FEATHER_DTYPE_F16 : FEATHER_DTYPE_BF16;
    a.causal = causal;
    a.scale = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(a.head_dim)));
    const hipStream_t stream = stream_of(q);
    const size_t bytes = feather_attention_workspace_size(&a);
    at::Tensor ws;
    if (bytes) ws = feather::workspace_for(q.device(), stream, bytes);
    check_status(feather_attention(&a, bytes ? ws.data_ptr() : nullptr, bytes ? static_cast<size_t>(ws.numel()) : 0, stream), what);
    return out;
}

at::Tensor attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal, std::optional<double> scale,
                     const OptTensor& k_lengths, const OptTensor& mask) {
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    check_attention(q, k, v, k_lengths, mask);
    check_scale(q, scale);
    const c10::DeviceGuard guard(q.device());
    feather_attention_args a{};
    a.batch = q.size(0);
    at::Tensor lengths, m;
    if (k_lengths.has_value() && q.size(0)) {
        lengths = k_lengths->contiguous();
        a.k_lengths = static_cast<const int32_t*>(lengths.data_ptr());
    }
    if (mask.has_value() && q.numel() && k.size(1)) {
        m = *mask;
        while (m.dim() < 4) m = m.unsqueeze(0);
        if (k.size(1) > 1 && (m.size(3) == 1 || m.stride(3) != 1)) {  // keys lie next to each other, shared dimensions stay so
            m = m.expand({m.size(0), m.size(1), m.size(2), k.size(1)}).clone(at::MemoryFormat::Contiguous);
        }
        a.mask = m.data_ptr();
        a.mask_dtype = m.scalar_type() == at::kBool ? FEATHER_DTYPE_BOOL : value_code(m.scalar_type(), "mask");
        a.mask_batch_stride = m.size(0) > 1 ? m.stride(0) : 0;
        a.mask_head_stride = m.size(1) > 1 ? m.stride(1) : 0;
        a.mask_query_stride = m.size(2) > 1 ? m.stride(2) : 0;
    }
    return run_attention(q, k, v, a, causal, scale, "attention");
}

at::Tensor packed_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& q_offsets,
                            const OptTensor& k_offsets, bool causal, std::optional<double> scale) {
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    check_packed_attention(q, k, v, q_offsets, k_offsets);
    check_scale(q, scale);
    const c10::DeviceGuard guard(q.device());
    const at::Tensor qo = q_offsets.contiguous(), ko = k_offsets.has_value() ? k_offsets->contiguous() : qo;
    feather_attention_args a{};
    a.batch = qo.size(0) - 1;
    a.q_offsets = static_cast<const int32_t*>(qo.data_ptr());
    a.k_offsets = static_cast<const int32_t*>(ko.data_ptr());
    return run_attention(q, k, v, a, causal, scale, "packed_attention");
}

// ---- fake tensors: the checks of the kernels above, and the results' shapes ----

at::Tensor like_meta(const at::Tensor& x) { return at::empty_symint(x.sym_sizes(), x.options()); }

at::Tensor rope_table_meta(const at::Tensor& positions, at::IntArrayRef axes, double theta, bool) {
    const int64_t pairs = check_table(positions, axes, theta);
    c10::SymDimVector shape(positions.sym_sizes().begin(), positions.sym_sizes().end());
    shape.back() = pairs;
    shape.push_back(2);
    return at::empty_symint(shape, positions.options().dtype(at::kFloat));
}
at::Tensor norm_rope_meta(const at::Tensor& x, const OptTensor& table, const OptTensor& weight, int64_t norm, double, bool) {
    check_rope(x, nullptr, table, weight, {}, norm);
    return like_meta(x);
}
std::tuple<at::Tensor, at::Tensor> qk_norm_rope_meta(const at::Tensor& q, const at::Tensor& k, const OptTensor& table,
                                                     const OptTensor& q_weight, const OptTensor& k_weight, int64_t norm, double,
                                                     bool) {
    check_rope(q, &k, table, q_weight, k_weight, norm);
    return {like_meta(q), like_meta(k)};
}
at::Tensor attention_meta(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool, std::optional<double> scale,
                          const OptTensor& k_lengths, const OptTensor& mask) {
    check_attention(q, k, v, k_lengths, mask);
    check_scale(q, scale);
    return like_meta(q);
}
at::Tensor packed_attention_meta(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& q_offsets,
                                 const OptTensor& k_offsets, bool, std::optional<double> scale) {
    check_packed_attention(q, k, v, q_offsets, k_offsets);
    check_scale(q, scale);
    return like_meta(q);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(feather_ops, m) {
    m.def("rope_table(Tensor positions, int[] axes, float theta, bool shared) -> Tensor");
    m.def("norm_rope(Tensor x, Tensor? table, Tensor? weight, int norm, float eps, bool halves) -> Tensor");
    m.def("qk_norm_rope(Tensor q, Tensor k, Tensor? table, Tensor? q_weight, Tensor? k_weight, int norm, float eps, "
          "bool halves) -> (Tensor, Tensor)");
    m.def("attention(Tensor q, Tensor k, Tensor v, bool causal, float? scale, Tensor? k_lengths, Tensor? mask) -> Tensor");
    m.def("packed_attention(Tensor q, Tensor k, Tensor v, Tensor q_offsets, Tensor? k_offsets, bool causal, float? scale) -> "
          "Tensor");
}

TORCH_LIBRARY_IMPL(feather_ops, CUDA, m) {
    m.impl("rope_table", &rope_table);
    m.impl("norm_rope", &norm_rope);
    m.impl("qk_norm_rope", &qk_norm_rope);
    m.impl("attention", &attention);
    m.impl("packed_attention", &packed_attention);
}

TORCH_LIBRARY_IMPL(feather_ops, Meta, m) {
    m.impl("rope_table", &rope_table_meta);
    m.impl("norm_rope", &norm_rope_meta);
    m.impl("qk_norm_rope", &qk_norm_rope_meta);
    m.impl("attention", &attention_meta);
    m.impl("packed_attention", &packed_attention_meta);
}
