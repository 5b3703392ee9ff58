// extern "C" entry points of rotary positions and attention (declared in
// include/featherops_amd.h). Sizes, types, strides and pointers are checked
// here, before anything is launched.
#include <cmath>

#include "attention.h"
#include "featherops_amd.h"
#include "rope.h"

namespace {

using namespace feather;

constexpr int64_t kMaxTokens = int64_t(1) << 30;
constexpr int64_t kMaxHeads = 1 << 16;
constexpr float kMaxScale = 0x1p127f;  // times log2(e) it is finite

bool value_type(int t) { return t == FEATHER_DTYPE_F16 || t == FEATHER_DTYPE_BF16 || t == FEATHER_DTYPE_F32; }
int round_up_pow2(int x) {
    int p = 1;
    while (p < x) p *= 2;
    return p;
}

// Rows are read 16 bytes at a time at 32-bit offsets within a tile of up to 64 of them.
bool strides_ok(int64_t batch, int64_t token, int64_t head) {
    return batch >= 0 && token >= 0 && head >= 0 && batch % 8 == 0 && token % 8 == 0 && head % 8 == 0 && token < (int64_t(1) << 23);
}
bool on_16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// FEATHER_OK with nothing to do leaves args->out untouched.
int attention_args(const feather_attention_args* a, AttnArgs& p, bool& empty) {
    if (!a || a->batch < 0 || a->batch > kAttnMaxBatch || a->q_tokens < 0 || a->q_tokens > kMaxTokens || a->k_tokens < 0 ||
        a->k_tokens > kMaxTokens || a->heads < 1 || a->heads > kMaxHeads || a->kv_heads < 1 || a->heads % a->kv_heads ||
        a->head_dim < 8 || a->head_dim > kAttnMaxDim || a->head_dim % 8 ||
        (a->dtype != FEATHER_DTYPE_F16 && a->dtype != FEATHER_DTYPE_BF16) || !(a->scale > 0.0f) || a->scale > kMaxScale ||
        (a->causal != 0 && a->causal != 1))
        return FEATHER_ERR_INVALID;
    // rows of a group of heads are counted in 32 bits
    if (a->q_tokens * (a->heads / a->kv_heads) > kMaxTokens) return FEATHER_ERR_INVALID;
    const bool packed = a->q_offsets || a->k_offsets;
    if (packed && (!a->q_offsets || !a->k_offsets || a->k_lengths || a->mask || a->batch < 1)) return FEATHER_ERR_INVALID;
    if (a->mask && a->mask_dtype != FEATHER_DTYPE_BOOL && a->mask_dtype != FEATHER_DTYPE_F32 && a->mask_dtype != a->dtype)
        return FEATHER_ERR_INVALID;
    empty = a->q_tokens == 0 || a->batch == 0;
    if (empty) return FEATHER_OK;
    if (!a->q || !a->out || !on_16(a->q) || !on_16(a->out) || !strides_ok(a->q_batch_stride, a->q_token_stride, a->q_head_stride))
        return FEATHER_ERR_INVALID;
    if (a->k_tokens > 0 &&
        (!a->k || !a->v || !on_16(a->k) || !on_16(a->v) || !strides_ok(a->k_batch_stride, a->k_token_stride, a->k_head_stride) ||
         !strides_ok(a->v_batch_stride, a->v_token_stride, a->v_head_stride)))
        return FEATHER_ERR_INVALID;
    if (a->mask && (a->mask_batch_stride < 0 || a->mask_head_stride < 0 || a->mask_query_stride < 0)) return FEATHER_ERR_INVALID;
    const int size = !a->mask ? 0 : a->mask_dtype == FEATHER_DTYPE_BOOL ? 1 : a->mask_dtype == FEATHER_DTYPE_F32 ? 4 : 2;
    if (size > 1 && reinterpret_cast<uintptr_t>(a->mask) % size) return FEATHER_ERR_INVALID;
    p.q = static_cast<const uint8_t*>(a->q);
    p.k = static_cast<const uint8_t*>(a->k);
    p.v = static_cast<const uint8_t*>(a->v);
    p.out = static_cast<uint16_t*>(a->out);
    p.mask = static_cast<const uint8_t*>(a->mask);
    p.q_offsets = a->q_offsets;
    p.k_offsets = a->k_offsets;
    p.k_lengths = a->k_lengths;
    p.q_batch = packed ? 0 : a->q_batch_stride * 2;
    p.q_row = a->q_token_stride * 2;
    p.q_head = a->q_head_stride * 2;
    p.k_batch = packed ? 0 : a->k_batch_stride * 2;
    p.k_row = a->k_token_stride * 2;
    p.k_head = a->k_head_stride * 2;
    p.v_batch = packed ? 0 : a->v_batch_stride * 2;
    p.v_row = a->v_token_stride * 2;
    p.v_head = a->v_head_stride * 2;
    p.mask_batch = a->mask_batch_stride * size;
    p.mask_head = a->mask_head_stride * size;
    p.mask_row = a->mask_query_stride * size;
    p.batch = static_cast<int>(a->batch);
    p.heads = static_cast<int>(a->heads);
    p.kv_heads = static_cast<int>(a->kv_heads);
    p.group = p.heads / p.kv_heads;
    p.dim = static_cast<int>(a->head_dim);
    p.sq = static_cast<int>(a->q_tokens);
    p.sk = static_cast<int>(a->k_tokens);
    p.mask_type = !a->mask ? kMaskNone : size == 1 ? kMaskBool : size == 2 ? kMaskHalf : kMaskF32;
    p.causal = a->causal;
    p.bf16 = a->dtype == FEATHER_DTYPE_BF16;
    p.scale = a->scale;
    return FEATHER_OK;
}

}  // namespace

extern "C" {

int feather_rope_table(const void* positions, int position_dtype, int64_t rows, const int* axis_dims, int axes, double theta,
                       int shared_ladder, float* table, hipStream_t stream) {
    if (position_dtype < FEATHER_POSITION_I32 || position_dtype > FEATHER_POSITION_F64 || rows < 0 || rows > kMaxTokens ||
        !axis_dims || axes < 1 || axes > kRopeMaxAxes || !(theta > 0.0) || !std::isfinite(theta))
        return FEATHER_ERR_INVALID;
    RopeTableArgs p{};
    for (int i = 0; i < axes; ++i) {
        if (axis_dims[i] < 0 || axis_dims[i] % 2 || axis_dims[i] > kRopeMaxDim) return FEATHER_ERR_INVALID;
        p.first[i + 1] = p.first[i] + axis_dims[i] / 2;
    }
    p.pairs = p.first[axes];
    if (p.pairs < 1 || p.pairs > kRopeMaxDim / 2) return FEATHER_ERR_INVALID;
    if (rows == 0) return FEATHER_OK;
    if (!positions || !table || reinterpret_cast<uintptr_t>(table) % 8) return FEATHER_ERR_INVALID;
    p.positions = positions;
    p.table = table;
    p.rows = rows;
    p.axes = axes;
    p.position_type = position_dtype;
    p.log_theta = std::log(theta);
    p.shared = shared_ladder != 0;
    return rope_table(p, stream);
}

int feather_qk_norm_rope(const feather_rope_args* a, hipStream_t stream) {
    if (!a || a->batch < 0 || a->tokens < 0 || a->tokens > kMaxTokens || a->batch > kMaxTokens || a->batch * a->tokens > kMaxTokens ||
        a->q_heads < 1 || a->q_heads > kMaxHeads || a->k_heads < 0 || a->k_heads > kMaxHeads || a->head_dim < 8 ||
        a->head_dim > kRopeMaxDim || a->head_dim % 8 || !value_type(a->dtype) ||
        (a->weight_dtype != a->dtype && a->weight_dtype != FEATHER_DTYPE_F32) || a->norm < kNoNorm || a->norm > kNormRow ||
        (a->pairs_of_halves != 0 && a->pairs_of_halves != 1))
        return FEATHER_ERR_INVALID;
    const int64_t most = a->q_heads > a->k_heads ? a->q_heads : a->k_heads;
    if (a->norm == kNormRow && most * round_up_pow2(static_cast<int>(a->head_dim)) > kRopeMaxRow) return FEATHER_ERR_INVALID;
    if (a->table && (a->pairs < 1 || a->pairs * 2 > a->head_dim || a->table_batch_stride < 0 || reinterpret_cast<uintptr_t>(a->table) % 4))
        return FEATHER_ERR_INVALID;
    if (a->norm == kNoNorm && (a->q_weight || a->k_weight)) return FEATHER_ERR_INVALID;
    if (a->batch * a->tokens == 0) return FEATHER_OK;
    if (!a->q || !a->q_out || (a->k_heads && (!a->k || !a->k_out))) return FEATHER_ERR_INVALID;
    const int size = a->dtype == FEATHER_DTYPE_F32 ? 4 : 2;
    RopeArgs p{};
    p.side[0] = {static_cast<const uint8_t*>(a->q), static_cast<uint8_t*>(a->q_out), a->q_weight, a->q_batch_stride * size,
                 a->q_token_stride * size, a->q_head_stride * size, static_cast<int>(a->q_heads)};
    p.side[1] = {static_cast<const uint8_t*>(a->k), static_cast<uint8_t*>(a->k_out), a->k_weight, a->k_batch_stride * size,
                 a->k_token_stride * size, a->k_head_stride * size, static_cast<int>(a->k_heads)};
    p.table = a->table;
    p.table_batch = a->table_batch_stride;
    p.tokens = a->batch * a->tokens;
    p.per_sample = static_cast<int>(a->tokens);
    p.dim = static_cast<int>(a->head_dim);
    p.pairs = static_cast<int>(a->pairs);
    p.type = a->dtype;
    p.weight_f32 = a->weight_dtype == FEATHER_DTYPE_F32;
    p.norm = a->norm;
    p.halves = a->pairs_of_halves;
    p.eps = a->eps;
    return qk_norm_rope(p, stream);
}

size_t feather_attention_workspace_size(const feather_attention_args* a) {
    AttnArgs p{};
    bool empty = false;
    return attention_args(a, p, empty) != FEATHER_OK || empty ? 0 : attention_plan(p).workspace;
}

int feather_attention_plan(const feather_attention_args* a, int64_t* plan) {
    if (!plan) return FEATHER_ERR_INVALID;
    AttnArgs p{};
    bool empty = false;
    const int status = attention_args(a, p, empty);
    plan[0] = plan[1] = plan[2] = 0;
    if (status != FEATHER_OK || empty) return status;
    const AttnPlan chosen = attention_plan(p);
    plan[0] = chosen.waves;
    plan[1] = chosen.splits;
    plan[2] = chosen.slots * (chosen.waves ? p.kv_heads : p.heads);
    return FEATHER_OK;
}

int feather_attention(const feather_attention_args* a, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    AttnArgs p{};
    bool empty = false;
    const int status = attention_args(a, p, empty);
    if (status != FEATHER_OK || empty) return status;
    AttnPlan plan = attention_plan(p);
    if (!workspace || workspace_bytes < plan.workspace) plan.splits = 1;
    return p.bf16 ? attention_bf16(p, plan, workspace, stream) : attention_f16(p, plan, workspace, stream);
}

}  // extern "C"
