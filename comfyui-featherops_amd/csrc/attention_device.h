// What the attention kernels share on the device: which rows and keys a workgroup works on, tiles
// of keys and values in LDS, and the products on them.
#pragma once

#include "attention.h"
#include "featherops_amd.h"
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
        job.b = p.by_blocks(slot);
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

// ---- a wave's 32 queries ----

template <int kMask>
constexpr int kMaskBytes = kMask == kMaskBool ? 1 : kMask == kMaskHalf ? 2 : 4;

// The mask's values for a wave's 32 queries and a tile's keys: lanes l and l + 32 load eight keys of the same query, l
// those of group 2 j, l + 32 of 2 j + 1. 16-bit values are loaded as the words that they lie in, and shifted into place when
// they are used: with 16-byte loads at addresses that are no multiples of 4, 2 x 1003 x 1003 x 16 heads of 64 took 35 us for 27, so
// 31 (8 bytes of a bool mask at any address cost less than this does).
template <bool kBf16, int kMask, int kKeyBlocks>
struct AttnMaskRegs {
    // values that are added to the scores: the scale comes before them
    static constexpr bool kAdds = kMask == kMaskHalf || kMask == kMaskF32;
    static constexpr int kWords = 2 * kMaskBytes<kMask>;                 // of eight values
    static constexpr bool kShifts = kMask == kMaskHalf;
    static constexpr int kLoaded = kShifts ? kWords + 1 : kWords;  // that they lie in
    uint32_t raw[kKeyBlocks][2][kLoaded];

    // those of the tile whose first key is key0, from the query's row; it has `keys` of them (what lies behind them is not read)
    __device__ __forceinline__ void load(const uint8_t* from, int key0, int keys) {
        if constexpr (kMask != kMaskNone) {
            const int skipped = kShifts ? static_cast<int>(reinterpret_cast<uintptr_t>(from) % 4) : 0;
            const bool any = kShifts && __any(skipped);
#pragma unroll
            for (int kb = 0; kb < kKeyBlocks; ++kb)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int key = key0 + kb * 32 + (2 * j + static_cast<int>(threadIdx.x) % 64 / 32) * 8;
                    const uint8_t* at = from - skipped + static_cast<int64_t>(key) * kMaskBytes<kMask>;
                    uint32_t(&w)[kLoaded] = raw[kb][j];
                    if (key0 + kKeyBlocks * 32 <= keys) {
                        __builtin_memcpy(w, kMask == kMaskBool ? at : __builtin_assume_aligned(at, 4), kWords * 4);
                        if (any) w[kLoaded - 1] = reinterpret_cast<const uint32_t*>(at)[skipped ? kLoaded - 1 : kWords - 1];
                    } else if constexpr (kMask == kMaskBool) {
#pragma unroll
                        for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (key + i < keys) w[i / 4] |= static_cast<uint32_t>(at[i]) << (8 * (i % 4));
                    } else {
                        const int bytes = skipped + (keys - key) * kMaskBytes<kMask>;
#pragma unroll
                        for (int i = 0; i < kLoaded; ++i) w[i] = key < keys && i * 4 < bytes ? reinterpret_cast<const uint32_t*>(at)[i] : 0;
                    }
                }
        }
    }
    // They are in their registers from here on.
    __device__ __forceinline__ void arrive() {
        if constexpr (kMask != kMaskNone) {
#pragma unroll
            for (int kb = 0; kb < kKeyBlocks; ++kb)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < kLoaded; ++i) asm volatile("" : "+v"(raw[kb][j][i]));
        }
    }
    __device__ __forceinline__ void put(f32x16 (&s)[kKeyBlocks], float scale, const uint8_t* from) {
        if constexpr (kMask != kMaskNone) {
            constexpr int kHalf = kWords / 2;  // words of four keys
            const uint32_t skipped = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from)) % 4 * 8;  // bits
#pragma unroll
            for (int kb = 0; kb < kKeyBlocks; ++kb)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t own[kWords];
#pragma unroll
                    for (int i = 0; i < kWords; ++i) {
                        if constexpr (kShifts) own[i] = __builtin_amdgcn_alignbit(raw[kb][j][i + 1], raw[kb][j][i], skipped);
                        else own[i] = raw[kb][j][i];
                    }
                    // lanes 32 apart trade four keys, so that each has four of both groups
                    uint32_t w[2][kHalf];
#pragma unroll
                    for (int i = 0; i < kHalf; ++i) {
                        const auto x = __builtin_amdgcn_permlane32_swap(own[i], own[kHalf + i], false, false);
                        w[0][i] = x[0];
                        w[1][i] = x[1];
                    }
#pragma unroll
                    for (int g = 0; g < 2; ++g)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int at = (2 * j + g) * 4 + e;
                            if constexpr (kMask == kMaskBool) {
                                s[kb][at] = (w[g][0] >> (8 * e)) & 0xff ? s[kb][at] : -INFINITY;
                            } else {
                                float add;
                                if constexpr (kMask == kMaskHalf) add = out_bits_to_f32<kBf16>(static_cast<uint16_t>(w[g][e / 2] >> (16 * (e % 2))));
                                else add = bits_f32(w[g][e]);
                                s[kb][at] = s[kb][at] * scale + add;
                            }
                        }
                }
        }
    }
};

// -inf for the tile's keys from `limit` on.
template <int kKeyBlocks>
__device__ __forceinline__ void attn_cut(f32x16 (&s)[kKeyBlocks], int key0, int limit) {
    const int first = key0 + static_cast<int>(threadIdx.x) % 64 / 32 * 4;
#pragma unroll
    for (int kb = 0; kb < kKeyBlocks; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (first + kb * 32 + e / 4 * 8 + e % 4 >= limit) s[kb][e] = -INFINITY;
}

// Where a lane reads in a tile: keys' chunk 2 s + lane / 32 of row lane % 32; values' four rows 4 (lane / 32) + i / 4 of
// block b's 32 columns, lane i of 16 giving four columns.
template <int kDim>
__device__ __forceinline__ void attn_lds_places(uint32_t keys, uint32_t values, uint32_t (&k_at)[kDim / 16], uint32_t (&v_at)[kDim / 32]) {
    const int lane = threadIdx.x % 64, l32 = lane % 32, half = lane / 32;
#pragma unroll
    for (int s = 0; s < kDim / 16; ++s) k_at[s] = keys + l32 * (kDim * 2) + ((2 * s + half) ^ swz_k<kDim>(l32)) * 16;
    const int i = lane % 16, r = 4 * half + i / 4;
#pragma unroll
    for (int b = 0; b < kDim / 32; ++b) {
        const int byte = b * 64 + (lane / 16 % 2) * 32 + (i % 4) * 8;
        v_at[b] = values + r * (kDim * 2) + ((byte / 16) ^ swz_v<kDim>(r)) * 16 + byte % 16;
    }
}

// Far below every score, but finite, and finite times the factor: a row that has seen nothing stays at weights 0.
template <bool kAdds>
__device__ __forceinline__ float kLowest(float factor) {
    return kAdds ? -3.402823466e38f : -8.0e37f / fmaxf(factor, 1.0f);
}

// One pass over the keys for 32 queries, a lane and the lane 32 away having one of them.
//
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T: a lane then has one query's
// column of scores, so maximum and sum run inside the lane, and the scores' registers, rounded to 16
// bits, are the second product's operand as they stand. The order of the 16 keys of an MFMA
// is free as long as both operands have it; V's is the one that the score layout leaves,
// which the transposing LDS read delivers. (Rounded weights are what 16-bit products take; their sum has them unrounded. bf16
// results are off by 2.3e-3 in the 2-norm with that, and by 1.7e-3 from their own rounding alone.) The maximum is replaced (and the
// sums scaled) only where a score exceeds it by more than 2^8: its value cancels in the result.
template <int kDim, bool kBf16, int kMask, int kKeyBlocks>
struct AttnWave {
    static constexpr int kSteps = kDim / 16, kBlocks = kDim / 32, kRowBytes = kDim * 2;
    static constexpr float kBias = kWeightBias<kBf16>;
    using Mask = AttnMaskRegs<kBf16, kMask, kKeyBlocks>;
    static constexpr bool kAdds = Mask::kAdds;

    u32x4 qf[kSteps];  // the queries: K Q^T's second operand
    uint32_t k_at[kSteps], v_at[kBlocks];
    f32x16 o[kBlocks];  // element 4 g + j of block b: column 32 b + 8 g + 4 (lane / 32) + j
    float factor, scale, top, total;
    Mask mask;
    const uint8_t* mask_row;

    // Tiles of keys lie at `keys` in LDS, of values at `values` (plus what scores() and add() are given).
    __device__ __forceinline__ void start(uint32_t keys, uint32_t values, float by) {
        attn_lds_places<kDim>(keys, values, k_at, v_at);
        scale = by;
        factor = kAdds ? kLog2e : by * kLog2e;
        top = kLowest<kAdds>(factor);
        total = 0.0f;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) o[b] = f32x16{};
    }

    __device__ __forceinline__ void scores(uint32_t stage, f32x16 (&s)[kKeyBlocks]) {
#pragma unroll
        for (int kb = 0; kb < kKeyBlocks; ++kb) s[kb] = f32x16{};
#pragma unroll
        for (int st = 0; st < kSteps; ++st)
#pragma unroll
            for (int kb = 0; kb < kKeyBlocks; ++kb)
                s[kb] = mfma32<kBf16>(lds_read16(k_at[st] + stage + kb * 32 * kRowBytes), qf[st], s[kb]);
    }

    // The mask's values on the scores, and -inf for keys from `limit` on where some of the tile's are (`cut`).
    __device__ __forceinline__ void masked(f32x16 (&s)[kKeyBlocks], int key0, int limit, bool cut) {
        mask.put(s, scale, mask_row);
        if (cut) attn_cut<kKeyBlocks>(s, key0, limit);
    }

    __device__ __forceinline__ void weights(f32x16 (&s)[kKeyBlocks], u32x4 (&pf)[2 * kKeyBlocks]) {
        float high = s[0][0];
#pragma unroll
        for (int kb = 0; kb < kKeyBlocks; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) high = fmaxf(high, s[kb][e]);
        high = max_halves(high);
        if (__any((high - top) * factor > kMaxLag)) {
            const float next = fmaxf(top, high);
            const float alpha = __builtin_amdgcn_exp2f((top - next) * factor);
            top = next;
            total *= alpha;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[b][e] *= alpha;
        }
        const float shift = kBias - top * factor;
#pragma unroll
        for (int kb = 0; kb < kKeyBlocks; ++kb)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                float w[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    w[j] = __builtin_amdgcn_exp2f(kAdds ? (s[kb][e + j] - top) * factor + kBias : s[kb][e + j] * factor + shift);
                    total += w[j];
                }
                pf[kb * 2 + e / 8][e % 8 / 2] = pack2<kBf16>(w[0], w[1]);
            }
    }

    __device__ __forceinline__ void add(uint32_t stage, const u32x4 (&pf)[2 * kKeyBlocks]) {
#pragma unroll
        for (int g = 0; g < 2 * kKeyBlocks; ++g)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const u32x2 lo = lds_read_transposed(v_at[b] + stage + g * 16 * kRowBytes);
                const u32x2 hi = lds_read_transposed(v_at[b] + stage + (g * 16 + 8) * kRowBytes);
                o[b] = mfma32<kBf16>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pf[g], o[b]);
            }
    }
};

}  // namespace feather
