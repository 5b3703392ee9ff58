// What the attention kernels share on the device: which rows and keys a workgroup works on, tiles
// of keys and values in LDS, and the products on them.
#pragma once

#include "attention.h"
#include "lds_dma.h"

namespace feather {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// ---- which rows, which keys ----

// Rows row0 .. of a sample's or sequence's `rows` (its first token is q_start, its keys are
// k_start .. k_start + keys).
struct AttnJob {
    int b, q_start, rows, k_start, keys, row0;
};

__device__ __forceinline__ int clamp_to(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// The slot-th block of kRows rows, a token counting as `per_token` rows; false past the last one.
// Packed: the sequences' blocks one after the other, found from their offsets by a sum over the
// lanes (64 sequences at a time). Tokens in front of the first and behind the last sequence
// count as sequences without keys, so their rows are written as zeros. Offsets are clamped to the
// tensors, so that none leads out of them.
template <int kRows>
__device__ __forceinline__ bool attn_job(const AttnArgs& p, int slot, int per_token, AttnJob& job) {
    if (!p.q_offsets) {
        const int blocks = (p.sq * per_token + kRows - 1) / kRows;
        job.b = slot / blocks;
        if (job.b >= p.batch) return false;
        job.row0 = (slot - job.b * blocks) * kRows;
        job.q_start = job.k_start = 0;
        job.rows = p.sq * per_token;
        job.keys = p.k_lengths ? clamp_to(p.k_lengths[job.b], 0, p.sk) : p.sk;
        return true;
    }
    const int lane = threadIdx.x % 64;
    int before = 0;
    for (int s0 = -1; s0 <= p.batch; s0 += 64) {
        const int s = s0 + lane;
        int start = 0, end = 0;
        if (s <= p.batch) {
            start = s < 0 ? 0 : clamp_to(p.q_offsets[s], 0, p.sq);
            end = s < p.batch ? clamp_to(p.q_offsets[s + 1], start, p.sq) : p.sq;
        }
        const int blocks = ((end - start) * per_token + kRows - 1) / kRows;
        int upto = blocks;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int other = __shfl_up(upto, d);
            if (lane >= d) upto += other;
        }
        const uint64_t past = __ballot(slot < before + upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            job.b = s0 + l;
            job.q_start = __builtin_amdgcn_readlane(start, l);
            job.rows = (__builtin_amdgcn_readlane(end, l) - job.q_start) * per_token;
            job.row0 = (slot - before - __builtin_amdgcn_readlane(upto - blocks, l)) * kRows;
            job.k_start = job.keys = 0;
            if (job.b >= 0 && job.b < p.batch) {
                job.k_start = clamp_to(p.k_offsets[job.b], 0, p.sk);
                job.keys = clamp_to(p.k_offsets[job.b + 1], job.k_start, p.sk) - job.k_start;
            }
            job.b = 0;  // (packed tensors have one batch stride, and masks are for samples)
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// ---- memory ----

// A buffer of `bytes` at p: reads past it give zeros, writes past it are dropped.
__device__ __forceinline__ i32x4 buffer_of(const void* p, int64_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const int n = bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : static_cast<int>(bytes);
    return i32x4{__builtin_amdgcn_readfirstlane(static_cast<int>(a)), __builtin_amdgcn_readfirstlane(static_cast<int>(a >> 32)),
                 __builtin_amdgcn_readfirstlane(n), 0x00027000};
}
constexpr uint32_t kPastEnd = 0x80000000u;  // an offset that no buffer_of() reaches

// 16 bytes a lane from the buffer into LDS at lds + 16 * lane; zeros past its end. (Inline asm for the reason
// given at dma16_lds.)
__device__ __forceinline__ void buffer_to_lds(i32x4 buffer, uint32_t offset, uint32_t lds) {
    asm volatile(
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %0, %1, 0 offen lds"
        :
        : "v"(offset), "s"(buffer), "{m0}"(lds)
        : "memory");
}

// The same for the compiler's own loads and stores.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource_of(const void* p, int64_t bytes) {
    const int n = bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : static_cast<int>(bytes);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, __builtin_amdgcn_readfirstlane(n), 0x00027000);
}

// ---- tiles in LDS ----
//
// A tile of keys or values is rows of kDim 16-bit values, as in memory, in chunks of 16 bytes;
// chunk c of row r sits at c ^ swz(r). Keys are read as operands of 32 rows, one chunk each: swz_k
// spreads a chunk of 8 or 16 rows over all banks. Values are read transposed, four rows by 64
// bytes for 32 lanes: swz_v puts the four rows next to each other. Rows of 192 bytes do that by themselves.
template <int kDim>
__device__ __forceinline__ int swz_k(int r) {
    if constexpr (kDim == 64) return swz(r);
    else if constexpr (kDim == 96) return (r >> 2) & 3;
    else return r & 15;
}
template <int kDim>
__device__ __forceinline__ int swz_v(int r) {
    if constexpr (kDim == 64) return ((r >> 1) & 1) << 2;
    else if constexpr (kDim == 96) return 0;
    else return (r & 3) << 2;
}

// Offsets in memory, from its first row, of what a lane copies of a tile of kKeys rows into LDS: instruction n of the tile
// writes 64 chunks, one a lane. Chunks past the head's own dimension read as zeros.
template <int kDim, bool kValues>
__device__ __forceinline__ uint32_t tile_offset(int n, int lane, int64_t row_bytes, int dim) {
    constexpr int kChunks = kDim / 8;
    const int id = n * 64 + lane, r = id / kChunks;
    const int c = (id - r * kChunks) ^ (kValues ? swz_v<kDim>(r) : swz_k<kDim>(r));
    return c * 8 < dim ? static_cast<uint32_t>(r * row_bytes) + c * 16 : kPastEnd;
}

typedef __attribute__((address_space(3))) const uint8_t* lds_ptr;

__device__ __forceinline__ u32x4 lds_read16(uint32_t at) {
    return *reinterpret_cast<__attribute__((address_space(3))) const u32x4*>(static_cast<uintptr_t>(at));
}
// Four rows of a 16-bit matrix, transposed: of each 16 lanes, lane i gives the address of four values of row i / 4 and
// gets the four rows' values of column i.
__device__ __forceinline__ u32x2 lds_read_transposed(uint32_t at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         reinterpret_cast<__attribute__((address_space(3))) i16x4*>(static_cast<uintptr_t>(at))));
}

// ---- products ----
// D (32x32) += A (32x16) * B (16x32). Lane l has row l % 32 of A and column l % 32 of B, each with 8
// values of the 16 (those of l / 32 = 0 and 1 follow one another), and of D column l % 32: element
// 4 g + j is row 8 g + 4 (l / 32) + j.
template <bool kBf16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (kBf16) {
        typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    }
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (kBf16) return f32x2_to_bf16x2_raw(a, b);
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, f16x2_t));
}

// The same value of the lane 32 away, combined.
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(f32_bits(x), f32_bits(x), false, false);
    return fmaxf(bits_f32(r[0]), bits_f32(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(f32_bits(x), f32_bits(x), false, false);
    return bits_f32(r[0]) + bits_f32(r[1]);
}

constexpr float kLog2e = 1.4426950408889634f;
// Weights are 2^(score - maximum + bias): fp16 ends at 2^-24 below, so its weights stand higher. They stay below
// 2^(8 + 7), as the maximum is let fall behind by up to 8.
template <bool kBf16>
constexpr float kWeightBias = kBf16 ? 0.0f : 7.0f;
constexpr float kMaxLag = 8.0f;

}  // namespace feather
