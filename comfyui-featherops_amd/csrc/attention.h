// Attention (attention_*.hip): arguments of the kernels and what the plan knows of them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace feather {

constexpr int kAttnMaxDim = 256;      // widest head
constexpr int kAttnMaxBatch = 65536;  // samples or packed sequences

// n / d for 0 <= n < 2^31, d > 0: with 2^shift >= d > 2^(shift - 1) and multiplier = ceil(2^(31 + shift) / d), 2 n * multiplier /
// 2^(32 + shift) is above n / d by less than n / 2^31 / d. (Five divisions by sizes took a workgroup 0.4 us before its
// first load.)
struct AttnDivisor {
    uint32_t multiplier, shift;
    static AttnDivisor of(int64_t d) {
        uint32_t shift = 0;
        while ((int64_t(1) << shift) < d) ++shift;
        return {static_cast<uint32_t>(((uint64_t(1) << (31 + shift)) + d - 1) / d), shift};
    }
    __device__ __forceinline__ int operator()(int n) const {
        return static_cast<int>(__umulhi(static_cast<uint32_t>(n) << 1, multiplier) >> shift);
    }
};

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
    // set at the launch: blocks of all samples, of one sample; heads of a class (tiles), heads that share a key head; rows:
    // workgroups that share keys, and what a store takes of a head
    AttnDivisor by_slots, by_blocks, by_class, by_group, by_splits, by_quads;
    int classes, class_heads;
};

// Which kernel takes a call, and how.
struct AttnPlan {
    int waves;      // attention_rows.h with 4 or 8 waves; 0: attention_tiles.h
    int64_t slots;  // blocks of rows, of one head or of one group of heads
    int splits;     // workgroups that share a block's keys, at most
    int least;      // tiles of 32 keys that one of them has at least
    size_t workspace;
};
constexpr size_t kAttnCounterBytes = 65536;
constexpr int kAttnMostSplits = 64;
AttnPlan attention_plan(const AttnArgs& p);

int attention_f16(const AttnArgs& p, const AttnPlan& plan, void* workspace, hipStream_t stream);
int attention_bf16(const AttnArgs& p, const AttnPlan& plan, void* workspace, hipStream_t stream);

}  // namespace feather
