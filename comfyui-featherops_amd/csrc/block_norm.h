// The norms around a block (block_norm.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace feather {

// Widest row: 1024 threads with two vectors of 8 values each (with four, the row's values, gates and
// affine vectors no longer fit the 128 registers of such a workgroup's threads).
constexpr int64_t kNormMaxCols = 16384;

struct NormArgs {
    const void* x;      // the residual stream (rows, cols), x_type
    int64_t x_stride;   // elements between rows
    const void* h;      // the block's output, y_type; null: the stream passes unchanged
    int64_t h_stride;
    // vectors of mod_f32 ? fp32 : y_type values; each may be null
    const void* gate;   // row r reads gate + r / gate_group * gate_stride
    int64_t gate_stride;
    const void* scale;  // row r reads scale + r / mod_group * scale_stride
    int64_t scale_stride;
    const void* shift;
    int64_t shift_stride;
    const void* post_weight;  // (cols,): h is normalised and weighted before the gate
    const void* weight;       // (cols,)
    const void* bias;         // (cols,)
    void* x_out;              // (rows, cols), x_type; unused without h
    void* y;                  // (rows, cols), y_type; null: codes and scales
    uint8_t* codes;           // packed MXFP4 operand
    uint8_t* scales;
    uint32_t gate_group, mod_group;  // at most `rows`
    int64_t rows;                    // below 2^31
    int cols;
    int x_type, y_type, mod_f32;  // MxType codes
    int layer;                    // 0: root mean square, 1: mean and variance
    float eps, residual_scale;
    int64_t row0;  // first row of this launch, a multiple of 128: set by block_norm
};

int block_norm(const NormArgs& p, hipStream_t stream);

}  // namespace feather
