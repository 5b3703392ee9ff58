// Attention over many queries: o = softmax(scale * q k^T + mask) v, one pass over the keys with a
// running maximum and sum.
//
// A wave holds 32 queries of one head, a workgroup of four 128; tiles of kKeys keys and values pass
// through a ring of two stages in LDS that all waves share, copied while the one before is worked on.
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T: a lane then has one query's
// column of scores, so maximum and sum run inside the lane, and the scores' registers, rounded to 16
// bits, are the second product's operand as they stand. The order of the 16 keys of an MFMA
// is free as long as both operands have it; V's is the one that the score layout leaves,
// which the transposing LDS read delivers. The maximum is replaced (and the sums scaled) only where
// a score exceeds it by more than 2^8: its value cancels in the result.
#pragma once

#include "attention_device.h"
#include "featherops_amd.h"

namespace feather {

template <int kDim>
struct AttnTile {
    static constexpr int kWaves = 4;
    static constexpr int kRows = 32 * kWaves;
    static constexpr int kKeys = kDim == 256 ? 32 : 64;
    static constexpr int kTileBytes = kKeys * kDim * 2;            // of keys or of values
    static constexpr int kCopies = kTileBytes / 1024 / kWaves;     // instructions a wave, for each of them
    static constexpr int kLds = 4 * kTileBytes;
};

// Four mask values of consecutive keys, of which the first n exist.
template <int kMask, bool kBf16>
__device__ __forceinline__ void mask4(const uint8_t* p, int n, float add[4]) {
    if (n <= 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) add[j] = 0.0f;
        return;
    }
    if constexpr (kMask == kMaskBool) {
        uint32_t w;
        if (n >= 4) {
            __builtin_memcpy(&w, p, 4);
        } else {
            w = p[0] | (n > 1 ? p[1] << 8 : 0) | (n > 2 ? p[2] << 16 : 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) add[j] = (w >> (8 * j)) & 0xff ? 0.0f : -INFINITY;
    } else if constexpr (kMask == kMaskHalf) {
        uint32_t w[2] = {0, 0};
        if (n >= 4) {
            __builtin_memcpy(w, p, 8);
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
            w[0] = h[0] | (n > 1 ? h[1] << 16 : 0);
            w[1] = n > 2 ? h[2] : 0;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) add[j] = out_bits_to_f32<kBf16>(static_cast<uint16_t>(w[j / 2] >> (16 * (j % 2))));
    } else {
        if (n >= 4) {
            __builtin_memcpy(add, p, 16);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) add[j] = j < n ? reinterpret_cast<const float*>(p)[j] : 0.0f;
        }
    }
}

template <int kDim, bool kBf16, int kMask>
__global__ __launch_bounds__(256, kDim <= 128 ? 2 : 1) void attention_tile_kernel(const AttnArgs p, int slots, int64_t per_xcd) {
    using T = AttnTile<kDim>;
    constexpr int kSteps = kDim / 16, kBlocks = kDim / 32, kKeyBlocks = T::kKeys / 32;
    constexpr int kRowBytes = kDim * 2;
    extern __shared__ __attribute__((aligned(1024))) uint8_t ring[];

    // workgroup i runs on XCD i % 8: each XCD takes consecutive blocks of few heads, whose keys its L2 keeps
    const int64_t id = static_cast<int64_t>(blockIdx.x % kNumXcd) * per_xcd + blockIdx.x / kNumXcd;
    const int head_slot = static_cast<int>(id / slots);
    if (blockIdx.x / kNumXcd >= per_xcd || head_slot >= p.heads) return;
    // (causal: the blocks with most keys first)
    const int slot = static_cast<int>(id - static_cast<int64_t>(head_slot) * slots);
    AttnJob job;
    if (!attn_job<T::kRows>(p, p.causal ? slots - 1 - slot : slot, 1, job)) return;
    const int head = head_slot, kv_head = head / p.group;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int l32 = lane % 32, half = lane / 32;
    const int row0 = job.row0 + wave * 32, row = row0 + l32;
    // keys [0, limit) are this lane's query's; [0, wg_keys) some query's of the workgroup
    const int shift = job.keys - job.rows;  // the last query sees all keys
    const int limit = p.causal ? min(job.keys, row + shift + 1) : job.keys;
    const int wave_keys = p.causal ? min(job.keys, row0 + 31 + shift + 1) : job.keys;
    const int wave_least = p.causal ? min(job.keys, row0 + shift + 1) : job.keys;
    const int wg_keys = p.causal ? min(job.keys, min(job.row0 + T::kRows, job.rows) + shift) : job.keys;
    const int tiles = wg_keys > 0 ? (wg_keys + T::kKeys - 1) / T::kKeys : 0;

    const uint8_t* k = p.k + job.b * p.k_batch + job.k_start * p.k_row + kv_head * p.k_head;
    const uint8_t* v = p.v + job.b * p.v_batch + job.k_start * p.v_row + kv_head * p.v_head;
    const uint32_t lds = lds_addr_of(ring);
    uint32_t k_off[T::kCopies], v_off[T::kCopies];
#pragma unroll
    for (int i = 0; i < T::kCopies; ++i) {
        k_off[i] = tile_offset<kDim, false>(wave * T::kCopies + i, lane, p.k_row, p.dim);
        v_off[i] = tile_offset<kDim, true>(wave * T::kCopies + i, lane, p.v_row, p.dim);
    }
    auto copy_tile = [&](int t) {
        const int key0 = t * T::kKeys;
        const int64_t rows_left = job.keys - key0 - 1;
        const i32x4 kb = buffer_of(k + key0 * p.k_row, rows_left * p.k_row + p.dim * 2);
        const i32x4 vb = buffer_of(v + key0 * p.v_row, rows_left * p.v_row + p.dim * 2);
        const uint32_t at = lds + (t & 1) * (2 * T::kTileBytes) + wave * (T::kCopies * 1024);
#pragma unroll
        for (int i = 0; i < T::kCopies; ++i) buffer_to_lds(kb, k_off[i], at + i * 1024);
#pragma unroll
        for (int i = 0; i < T::kCopies; ++i) buffer_to_lds(vb, v_off[i], at + T::kTileBytes + i * 1024);
    };
    if (tiles) copy_tile(0);

    // queries: the second operand of K Q^T, kept in registers
    u32x4 qf[kSteps];
    {
        const uint8_t* q = p.q + job.b * p.q_batch + (job.q_start + static_cast<int64_t>(row0)) * p.q_row + head * p.q_head;
        const auto qb = resource_of(q, (job.rows - row0 - 1) * p.q_row + p.dim * 2);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int d = s * 16 + half * 8;
            qf[s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                  qb, d < p.dim ? static_cast<uint32_t>(l32 * p.q_row) + d * 2 : kPastEnd, 0, 0));
        }
    }

    // where in a tile this lane reads: keys' chunk 2 s + half of row l32; values' four rows 4 half + i / 4 of
    // block b's 32 columns, lane i of 16 giving four columns
    uint32_t k_at[kSteps], v_at[kBlocks];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) k_at[s] = lds + l32 * kRowBytes + ((2 * s + half) ^ swz_k<kDim>(l32)) * 16;
    {
        const int i = lane % 16, r = 4 * half + i / 4;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const int byte = b * 64 + (lane / 16 % 2) * 32 + (i % 4) * 8;
            v_at[b] = lds + T::kTileBytes + r * kRowBytes + ((byte / 16) ^ swz_v<kDim>(r)) * 16 + byte % 16;
        }
    }

    const float factor = kMask ? kLog2e : p.scale * kLog2e;
    constexpr float kBias = kWeightBias<kBf16>;
    // far below every score, but finite, and finite times the factor: a row that has seen nothing stays at weights 0
    float top = kMask ? -3.402823466e38f : -8.0e37f / fmaxf(factor, 1.0f);
    float total = 0.0f;
    f32x16 o[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) o[b] = f32x16{};
    const uint8_t* mask = nullptr;
    if constexpr (kMask != kMaskNone)
        mask = p.mask + job.b * p.mask_batch + head * p.mask_head + min(row, job.rows - 1) * p.mask_row;

    for (int t = 0; t < tiles; ++t) {
        // this wave's copies of tile t have landed and its reads of the other stage are done; then everyone's
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (t + 1 < tiles) copy_tile(t + 1);
        const int key0 = t * T::kKeys;
        if (key0 >= wave_keys) continue;
        const uint32_t stage = (t & 1) * (2 * T::kTileBytes);

        f32x16 s[kKeyBlocks];
#pragma unroll
        for (int kb = 0; kb < kKeyBlocks; ++kb) s[kb] = f32x16{};
#pragma unroll
        for (int st = 0; st < kSteps; ++st)
#pragma unroll
            for (int kb = 0; kb < kKeyBlocks; ++kb)
                s[kb] = mfma32<kBf16>(lds_read16(k_at[st] + stage + kb * 32 * kRowBytes), qf[st], s[kb]);

        if constexpr (kMask != kMaskNone) {
#pragma unroll
            for (int kb = 0; kb < kKeyBlocks; ++kb)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int key = key0 + kb * 32 + g * 8 + half * 4;
                    constexpr int kSize = kMask == kMaskBool ? 1 : kMask == kMaskHalf ? 2 : 4;
                    float add[4];
                    mask4<kMask, kBf16>(mask + static_cast<int64_t>(key) * kSize, job.keys - key, add);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[kb][g * 4 + j] = s[kb][g * 4 + j] * p.scale + add[j];
                }
        }
        if (key0 + T::kKeys > wave_least) {
#pragma unroll
            for (int kb = 0; kb < kKeyBlocks; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = key0 + kb * 32 + (e / 4) * 8 + half * 4 + e % 4;
                    if (key >= limit) s[kb][e] = -INFINITY;
                }
        }

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
        const float shift_by = kBias - top * factor;
        u32x4 pf[2 * kKeyBlocks];
#pragma unroll
        for (int kb = 0; kb < kKeyBlocks; ++kb)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                float w[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    w[j] = __builtin_amdgcn_exp2f(kMask ? (s[kb][e + j] - top) * factor + kBias
                                                        : s[kb][e + j] * factor + shift_by);
                    total += w[j];
                }
                pf[kb * 2 + e / 8][e % 8 / 2] = pack2<kBf16>(w[0], w[1]);
            }

#pragma unroll
        for (int g = 0; g < 2 * kKeyBlocks; ++g)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const u32x2 lo = lds_read_transposed(v_at[b] + stage + g * 16 * kRowBytes);
                const u32x2 hi = lds_read_transposed(v_at[b] + stage + (g * 16 + 8) * kRowBytes);
                o[b] = mfma32<kBf16>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pf[g], o[b]);
            }
    }

    total = sum_halves(total);
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    // element 4 g + j of block b is column 32 b + 8 g + 4 half + j: lanes 32 apart trade four columns, so that each
    // stores eight
    uint16_t* out = p.out + ((static_cast<int64_t>(job.b) * p.sq + job.q_start + row0) * p.heads + head) * p.dim;
    const int64_t out_row = static_cast<int64_t>(p.heads) * p.dim * 2;
    const auto ob = resource_of(out, (job.rows - row0 - 1) * out_row + p.dim * 2);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
            uint32_t w[2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    w[i][j] = pack2<kBf16>(o[b][(g + i) * 4 + j * 2] * inverse, o[b][(g + i) * 4 + j * 2 + 1] * inverse);
            const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
            const int d = b * 32 + (g + half) * 8;
            __builtin_amdgcn_raw_buffer_store_b128(u32x4{x[0], y[0], x[1], y[1]}, ob,
                                                   d < p.dim ? static_cast<uint32_t>(l32 * out_row) + d * 2 : kPastEnd, 0, 0);
        }
}

template <int kDim, bool kBf16, int kMask>
int launch_attention_tiles(const AttnArgs& p, hipStream_t stream) {
    using T = AttnTile<kDim>;
    const int64_t slots = p.q_offsets ? p.sq / T::kRows + p.batch + 2
                                      : static_cast<int64_t>(p.batch) * ((p.sq + T::kRows - 1) / T::kRows);
    const int64_t per_xcd = (slots * p.heads + kNumXcd - 1) / kNumXcd;
    if (slots > 0x7fffffff || per_xcd * kNumXcd * 256 > 0xffffffffll) return FEATHER_ERR_UNSUPPORTED;
    auto* kernel = attention_tile_kernel<kDim, kBf16, kMask>;
    kernel<<<dim3(static_cast<uint32_t>(per_xcd * kNumXcd)), 256, T::kLds, stream>>>(p, static_cast<int>(slots), per_xcd);
    return hipGetLastError() == hipSuccess ? FEATHER_OK : FEATHER_ERR_LAUNCH;
}

template <int kDim, bool kBf16>
int attention_tiles_mask(const AttnArgs& p, hipStream_t stream) {
    switch (p.mask_type) {
        case kMaskNone: return launch_attention_tiles<kDim, kBf16, kMaskNone>(p, stream);
        case kMaskBool: return launch_attention_tiles<kDim, kBf16, kMaskBool>(p, stream);
        case kMaskHalf: return launch_attention_tiles<kDim, kBf16, kMaskHalf>(p, stream);
        default: return launch_attention_tiles<kDim, kBf16, kMaskF32>(p, stream);
    }
}

template <bool kBf16>
int attention_tiles(const AttnArgs& p, hipStream_t stream) {
    if (p.dim <= 64) return attention_tiles_mask<64, kBf16>(p, stream);
    if (p.dim <= 96) return attention_tiles_mask<96, kBf16>(p, stream);
    if (p.dim <= 128) return attention_tiles_mask<128, kBf16>(p, stream);
    return attention_tiles_mask<256, kBf16>(p, stream);
}

}  // namespace feather
