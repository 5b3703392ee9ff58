// Attention (attention_*.hip): arguments of the kernels and what the plan knows of them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace feather {

constexpr int kAttnMaxDim = 256;      // widest head
constexpr int kAttnMaxBatch = 65536;  // samples or packed sequences

enum AttnMask { kMaskNone = 0, kMaskBool = 1, kMaskHalf = 2, kMaskF32 = 3 };

struct AttnArgs {
    const uint8_t* q;  // 16-bit values; strides in bytes, the head dimension contiguous
    const uint8_t* k;
    const uint8_t* v;
    uint16_t* out;  // (rows, heads, dim) contiguous
    const uint8_t* mask;
    const int* q_offsets;  // packed sequences: batch + 1 each; null: samples of one size
    const int* k_offsets;
    const int* k_lengths;  // (batch,) or null
    int64_t q_batch, q_row, q_head;
    int64_t k_batch, k_row, k_head;
    int64_t v_batch, v_row, v_head;
    int64_t mask_batch, mask_head, mask_row;  // bytes; 0 where the mask is shared
    int batch, heads, kv_heads, group, dim;
    int sq, sk;  // tokens of a sample; packed: all tokens
    int mask_type, causal, bf16;
    float scale;
};

int attention_tiles_f16(const AttnArgs& p, hipStream_t stream);
int attention_tiles_bf16(const AttnArgs& p, hipStream_t stream);

}  // namespace feather
