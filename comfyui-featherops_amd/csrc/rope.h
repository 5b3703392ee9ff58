// Rotary positions and the norm of queries and keys (rope.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace feather {

constexpr int kRopeMaxAxes = 8;
constexpr int kRopeMaxDim = 256;
// norm over a row: heads times the head's size, the latter rounded up to a power of two
constexpr int64_t kRopeMaxRow = 16384;

struct RopeTableArgs {
    const void* positions;  // (rows, axes)
    float* table;           // (rows, pairs, 2)
    int64_t rows;
    int pairs, axes, position_type;  // 0 int32, 1 int64, 2 fp32, 3 fp64
    int first[kRopeMaxAxes + 1];     // an axis's first pair; the last one's end
    double log_theta;
    int shared;
};

struct RopeSide {
    const uint8_t* x;  // strides in bytes
    uint8_t* out;      // contiguous
    const void* weight;
    int64_t batch_stride, token_stride, head_stride;
    int heads;
};

struct RopeArgs {
    RopeSide side[2];    // queries, keys (no heads: none)
    const float* table;  // null: positions are left as they are
    int64_t table_batch;  // floats; 0 where all samples share the table
    int64_t tokens;      // of all samples
    int per_sample, dim, pairs, type, weight_f32, norm, halves;
    float eps;
};

enum RopeNorm { kNoNorm = 0, kNormHead = 1, kNormRow = 2 };

int rope_table(const RopeTableArgs& p, hipStream_t stream);
int qk_norm_rope(const RopeArgs& p, hipStream_t stream);

}  // namespace feather
