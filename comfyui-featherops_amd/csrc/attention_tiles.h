// Attention over many queries: o = softmax(scale * q k^T + mask) v, one pass over the keys with a
// running maximum and sum.
//
// A wave holds 32 queries of one head, a workgroup of four 128. Keys and values pass through two
// rings of units of 32 keys in LDS that all waves share; two waves copy keys, two copy values, several
// units ahead. In its turn u a wave makes the weights of unit u from its scores, which is work for the vector
// units, and beside it runs the products that give the scores of unit u + 1 and that add the values of
// unit u - 1: the instructions of both stand alternately in the code, since a wave issues them in order and the
// second of two products would hold up whatever stands behind it. (With the products of a unit first and
// its weights behind them, 32760 x 32760 x 12 heads of 128 took 7.0 ms: the two overlapped only between the two waves of
// a SIMD.)
//
// Now 5.8 to 5.95 ms (1.11 to 1.13 PFLOP/s; 1.02 at 4096 x 4096 x 24 heads of 128, 1.05 at 8192 x 8192 x 12 of 256): by the counters
// matrix units busy 65% of the cycles (49 and 45%) at the 1.6 GHz that the card holds under it (1.9 and 2.0), no LDS bank conflicts, LDS
// reads active in 32% (25 and 22), waves waiting 24% of theirs (28 and 34): what does not fall side by side in two waves a SIMD waits.
// Over 512 keys, 2 x 8190 x 40 heads: 250 us with a key mask, 690 TFLOP/s, of which a workgroup's start, its queries' load and its
// stores take 100, as they overlap with the other workgroup of the CU alone (LDS and registers hold two); 226 without a mask.
// Numbers of keys that are no multiple of 32 cost a bool mask the loads of its last bytes, one by one: 77 keys 155 us, 96 keys 137.
// 32 queries a wave: with 64 each key read from LDS served twice the products, but scores and results of both left no
// registers to keep products and weights apart. Two teams of waves that take half the keys each were faster nowhere.
//
// The products are taken transposed, as in AttnWave. They are inline asm, which keeps their order and their
// accumulators' place: results in accumulation registers where the vector registers do not hold everything.
#pragma once

#include "attention_device.h"

namespace feather {

template <int kDim, int kMask>
struct AttnTile {
    static constexpr int kWaves = 4;
    static constexpr int kRows = 32 * kWaves;
    static constexpr int kUnitBytes = 32 * kDim * 2;  // of keys or of values
    static constexpr int kCopies = kUnitBytes / 2048;  // instructions of each of two waves
    static constexpr int kRing = 4;                    // units in each ring
    // Units that are copied at once, and turns between barriers. A mask's values are loaded by the compiler's own loads,
    // whose waits, as it knows of no copies, are waits for all copies before them: so two turns apart.
    static constexpr int kBatch = kMask == kMaskNone ? 1 : 2;
    static constexpr int kLds = 2 * kRing * kUnitBytes;
    static constexpr bool kAccumulation = kDim == 256;  // results in accumulation registers
};

// Their hazards are the code's own business: a source that another vector instruction wrote needs two wait states before
// the product (kPadded puts them there), whoever else reads a result waits for it.
#define FEATHER_MFMA32(type, before, result, from) \
    asm volatile(before "v_mfma_f32_32x32x16_" type " %0, %1, %2, " from : result(c) : "v"(a), "v"(b))
template <bool kBf16>
__device__ __forceinline__ void mfma_first(f32x16& c, u32x4 a, u32x4 b) {
    if constexpr (kBf16) FEATHER_MFMA32("bf16", "s_nop 1\n\t", "=&v", "0");
    else FEATHER_MFMA32("f16", "s_nop 1\n\t", "=&v", "0");
}
template <bool kBf16, bool kAccumulation, bool kPadded>
__device__ __forceinline__ void mfma_next(f32x16& c, u32x4 a, u32x4 b) {
    if constexpr (kAccumulation) {
        if constexpr (kBf16) FEATHER_MFMA32("bf16", "s_nop 1\n\t", "+a", "%0");
        else FEATHER_MFMA32("f16", "s_nop 1\n\t", "+a", "%0");
    } else if constexpr (kPadded) {
        if constexpr (kBf16) FEATHER_MFMA32("bf16", "s_nop 1\n\t", "+v", "%0");
        else FEATHER_MFMA32("f16", "s_nop 1\n\t", "+v", "%0");
    } else {
        if constexpr (kBf16) FEATHER_MFMA32("bf16", "", "+v", "%0");
        else FEATHER_MFMA32("f16", "", "+v", "%0");
    }
}
#undef FEATHER_MFMA32
// Until an accumulator's values are in its registers: reads of them stay behind.
template <bool kAccumulation = false>
__device__ __forceinline__ void settle(f32x16& c) {
    if constexpr (kAccumulation) asm volatile("s_nop 15\n\ts_nop 3" : "+a"(c));
    else asm volatile("s_nop 15\n\ts_nop 3" : "+v"(c));
}

template <int kDim, bool kBf16, int kMask>
__global__ __launch_bounds__(256, kDim > 128 ? 1 : kDim == 64 && kMask == kMaskNone ? 4 : 2) void attention_tile_kernel(
    const AttnArgs p, int slots, int per_xcd) {
    using T = AttnTile<kDim, kMask>;
    using Mask = AttnMaskRegs<kBf16, kMask, 1>;
    constexpr int kSteps = kDim / 16, kBlocks = kDim / 32, kRowBytes = kDim * 2;
    constexpr bool kAdds = Mask::kAdds;
    constexpr float kBias = kWeightBias<kBf16>;
    __shared__ __attribute__((aligned(1024))) uint8_t rings[T::kLds];

    // Workgroup i runs on XCD i % 8. Where all blocks have the same keys to do, each XCD takes consecutive blocks of few heads, whose
    // keys its L2 keeps. Where they have not (causal, packed, lengths), an XCD has a class of heads, or a share of one (as many
    // classes as the largest power of two that divides the heads, up to 8), and takes the blocks of all its heads in
    // turn, causal ones with most keys first: the work is alike on all XCDs, and what is left for the end is small. (4096 x 4096, causal,
    // 32 heads over 8: 172 us with a head behind the other, so 154; 8192: 536 and 518; sequences of 0 to 512, 28 heads: 23.7
    // and 20.0. Blocks alike, 2 x 8190 x 512 x 40 heads: 2% slower so.)
    int head, slot;
    const int xcd = static_cast<int>(blockIdx.x % kNumXcd), nth = static_cast<int>(blockIdx.x / kNumXcd);
    if (p.causal || p.q_offsets || p.k_lengths) {
        const int item = nth * (kNumXcd / p.classes) + xcd / p.classes, behind = p.by_class(item);
        head = xcd % p.classes * p.class_heads + item - behind * p.class_heads;
        slot = p.causal ? slots - 1 - behind : behind;
        if (behind >= slots) return;
    } else {
        const int id = xcd * per_xcd + nth;
        head = p.by_slots(id);
        slot = id - head * slots;
        if (head >= p.heads) return;
    }
    AttnJob job;
    if (!attn_job<T::kRows>(p, slot, 1, job)) return;
    const int kv_head = p.by_group(head);

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int l32 = lane % 32, half = lane / 32;
    const int row0 = job.row0 + wave * 32;
    // The last query sees all keys. Keys [0, limit) are this lane's query's, and the wave's queries see wave_keys at most and
    // wave_least at least.
    const int shift = job.keys - job.rows;
    const int limit = p.causal ? min(job.keys, row0 + l32 + shift + 1) : job.keys;
    const int wave_keys = row0 >= job.rows ? 0 : p.causal ? min(job.keys, row0 + 32 + shift) : job.keys;
    const int wave_least = p.causal ? min(job.keys, row0 + shift + 1) : job.keys;
    const int wg_keys = p.causal ? min(job.keys, min(job.row0 + T::kRows, job.rows) + shift) : job.keys;
    // units, in twos; two at least, of which a wave without keys sees none. All waves pass the barriers of wg_units turns, the
    // most that one of them has.
    const int units = max(1, (wave_keys + 63) / 64) * 2, wg_units = max(1, (wg_keys + 63) / 64) * 2;

    // waves 0 and 1 copy keys, 2 and 3 values
    const bool copies_keys = wave < 2;
    const int64_t copy_row = copies_keys ? p.k_row : p.v_row;
    const uint8_t* copy_from = copies_keys ? p.k + job.b * p.k_batch + job.k_start * p.k_row + kv_head * p.k_head
                                           : p.v + job.b * p.v_batch + job.k_start * p.v_row + kv_head * p.v_head;
    const uint32_t lds_k = lds_addr_of(rings), lds_v = lds_k + T::kRing * T::kUnitBytes;
    const uint32_t copy_to = (copies_keys ? lds_k : lds_v) + wave % 2 * (T::kCopies * 1024);
    uint32_t copy_off[T::kCopies];
#pragma unroll
    for (int i = 0; i < T::kCopies; ++i)
        copy_off[i] = copies_keys ? tile_offset<kDim, false>(wave % 2 * T::kCopies + i, lane, copy_row, p.dim)
                                  : tile_offset<kDim, true>(wave % 2 * T::kCopies + i, lane, copy_row, p.dim);
    auto copy_unit = [&](int u) {  // (past the last key: zeros)
        const int64_t key0 = u * 32;
        const i32x4 b = buffer_of(copy_from + key0 * copy_row, key0 < job.keys ? (job.keys - key0 - 1) * copy_row + p.dim * 2 : 0);
        const uint32_t at = copy_to + u % T::kRing * T::kUnitBytes;
#pragma unroll
        for (int i = 0; i < T::kCopies; ++i) buffer_to_lds(b, copy_off[i], at + i * 1024);
    };
    // What is copied before turn u: keys up to u + kRing, in the place of those that turn u - 1 has read last, and values up
    // to u + kRing - 2 likewise.
    const int ahead = copies_keys ? T::kRing : T::kRing - 2;
    // Before turn u, the first one too (unit 0's keys have been read by then): what it and the kBatch - 1 behind it read of
    // this wave's copies has landed (one turn at a time: all but the last unit's), and its reads of what is copied over
    // next are done; then everyone's.
    auto wait_batch = [&] {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(T::kBatch == 1 ? T::kCopies : 0) : "memory");
    };
    auto copy_batch = [&](int u) {
#pragma unroll
        for (int i = 1 - T::kBatch; i <= 0; ++i) copy_unit(u + ahead + i);
    };
    for (int u = 0; u <= ahead - T::kBatch; ++u) copy_unit(u);

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
    uint32_t k_at[kSteps], v_at[kBlocks];
    attn_lds_places<kDim>(lds_k, lds_v, k_at, v_at);
    // masks of two units each: what a turn cuts with was loaded two turns before (fp32 masks, which are too wide for that,
    // in the turn before)
    constexpr int kSets = kMask == kMaskF32 ? 1 : 2;
    Mask mask[kSets][2];
    const uint8_t* mask_row = nullptr;
    if constexpr (kMask != kMaskNone)
        mask_row = p.mask + job.b * p.mask_batch + head * p.mask_head + min(row0 + l32, job.rows - 1) * p.mask_row;
    const float factor = kAdds ? kLog2e : p.scale * kLog2e;
    float top = kLowest<kAdds>(factor), by, total = 0.0f;
    f32x16 o[kBlocks], s0[1], s1[1];  // results; scores of even and odd units
    u32x4 p0[2], p1[2];               // their weights
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) o[b] = f32x16{};
    p1[0] = p1[1] = u32x4{};
    auto read_k = [&](int s, uint32_t at) { return lds_read16(k_at[s] + at); };
    auto read_v = [&](int n, uint32_t at) {  // block n % kBlocks of 16 keys
        const uint32_t from = v_at[n % kBlocks] + at + n / kBlocks * 16 * kRowBytes;
        const u32x2 lo = lds_read_transposed(from), hi = lds_read_transposed(from + 8 * kRowBytes);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    // the mask on unit u's scores, and what a query does not see of it
    auto cut = [&](f32x16 (&s)[1], Mask& mask, int u) {
        const bool past = u * 32 + 32 > wave_least;
        if (kMask != kMaskNone || past) settle(s[0]);
        mask.put(s, p.scale, mask_row);
        if (past) attn_cut<1>(s, u * 32, limit);
    };
    auto load_masks = [&](Mask (&m)[2], int u) {
#pragma unroll
        for (int i = 0; i < 2; ++i) m[i].load(mask_row, (u + i) * 32, job.keys);
    };
    // Unit u: its weights from its scores `now`; beside that the products that give the scores of the unit ahead, whose keys
    // are at ka, and that add the unit before with its weights `old` and values at va. The keys of the unit after
    // that are at kn. high: the scores' maximum, of `now` on the way in, of `next` on the way out.
    u32x4 kf[3];
    float high;
    auto turn = [&](int u, f32x16 (&now)[1], f32x16 (&next)[1], u32x4 (&pf)[2], u32x4 (&old)[2], uint32_t ka, uint32_t va, uint32_t kn, Mask& its_mask,
                    bool first, bool last) {
        // (whether the turn begins a batch, with copies and after a barrier before which nothing is read ahead; whether it ends one)
        // A maximum that has fallen behind is raised, by a power of two of the weights: that leaves the rounded ones of the unit
        // before, which are still to be added, as exact as they were. (A row that had seen nothing starts anew.)
        const float behind = (high - top) * factor;
        if (__any(behind > kMaxLag)) {
            const float steps = behind > 0.0f ? ceilf(behind) : 0.0f;
            const bool anew = steps > 512.0f;
            const float alpha = anew ? 0.0f : __builtin_amdgcn_ldexpf(1.0f, -static_cast<int>(steps));
            top = anew ? high : top + steps / factor;
            by = kBias - top * factor;
            total *= alpha;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                settle<T::kAccumulation>(o[b]);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[b][e] *= alpha;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w = old[i / 4][i % 4];
                old[i / 4][i % 4] = pack2<kBf16>(out_bits_to_f32<kBf16>(static_cast<uint16_t>(w)) * alpha,
                                                 out_bits_to_f32<kBf16>(static_cast<uint16_t>(w >> 16)) * alpha);
            }
        }
        // Two scores to weights, in two steps a product apart; the first product has the copies beside it.
        float w[2];
        auto beside = [&](int slot) {
#pragma unroll
            for (int h = (slot - 1) * 16 / (2 * kSteps - 1); h < slot * 16 / (2 * kSteps - 1); ++h) {
                const int e = h / 2 * 2;
                if (h % 2 == 0) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        w[j] = __builtin_amdgcn_exp2f(kAdds ? (now[0][e + j] - top) * factor + kBias : now[0][e + j] * factor + by);
                } else {
                    total += w[0];
                    total += w[1];
                    uint32_t both = pack2<kBf16>(w[0], w[1]);
                    asm volatile("" : "+v"(both), "+v"(total));  // (here, not where they are used)
                    pf[e / 8][e % 8 / 2] = both;
                }
            }
        };
        u32x4 vf[3];
        static_assert(kSteps == 2 * kBlocks);
        if (T::kBatch > 1 && first) {
            kf[0] = read_k(0, ka);
            kf[1] = read_k(1, ka);
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (s + 2 < kSteps) kf[(s + 2) % 3] = read_k(s + 2, ka);
            else vf[s + 2 - kSteps] = read_v(s + 2 - kSteps, va);
            __builtin_amdgcn_sched_barrier(0);
            if (s == 0) mfma_first<kBf16>(next[0], kf[0], qf[0]);
            else mfma_next<kBf16, false, T::kAccumulation>(next[0], kf[s % 3], qf[s]);
            __builtin_amdgcn_sched_barrier(0);
            if (s) beside(s);
            else if (first) copy_batch(u);
        }
        __builtin_amdgcn_sched_barrier(0);
        cut(next, its_mask, u + 1);
        if (kMask != kMaskNone && kSets == 1 && last) load_masks(mask[0], u + 2);
        high = -INFINITY;
#pragma unroll
        for (int n = 0; n < kSteps; ++n) {
            if (n + 2 < kSteps) vf[(n + 2) % 3] = read_v(n + 2, va);
            else if (T::kBatch == 1 || !last) kf[n + 2 - kSteps] = read_k(n + 2 - kSteps, kn);
            __builtin_amdgcn_sched_barrier(0);
            mfma_next<kBf16, T::kAccumulation, T::kAccumulation>(o[n % kBlocks], vf[n % 3], old[n / kBlocks]);
            __builtin_amdgcn_sched_barrier(0);
            beside(kSteps + n);
            // (the scores have settled: half of the products later)
            constexpr int kFrom = kSteps / 2;
            if (n >= kFrom) {
#pragma unroll
                for (int e = (n - kFrom) * 8 / kFrom * 2; e < (n - kFrom + 1) * 8 / kFrom * 2; e += 2)
                    high = fmaxf(fmaxf(high, next[0][e]), next[0][e + 1]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        high = max_halves(high);
    };

    // Unit 0 has none before it: weights of zero, and values of zero in the place that is copied to last.
    for (int i = threadIdx.x; i < T::kUnitBytes / 16; i += 256)
        reinterpret_cast<u32x4*>(rings + (2 * T::kRing - 1) * T::kUnitBytes)[i] = u32x4{};
    // Units 0 to 2 of the keys and 0 of the values have landed.
    Mask mask0;
    mask0.load(mask_row, 0, job.keys);
    load_masks(mask[0], 1);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(T::kBatch == 1 ? T::kCopies : 0) : "memory");
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        if (s == 0) mfma_first<kBf16>(s0[0], read_k(0, 0), qf[0]);
        else mfma_next<kBf16, false, true>(s0[0], read_k(s, 0), qf[s]);
    }
    if (T::kBatch == 1) {
        kf[0] = read_k(0, T::kUnitBytes);
        kf[1] = read_k(1, T::kUnitBytes);
    }
    if (kMask == kMaskNone) settle(s0[0]);
    cut(s0, mask0, 0);
    high = top;
#pragma unroll
    for (int e = 0; e < 16; ++e) high = fmaxf(high, s0[0][e]);
    top = high = max_halves(high);
    by = kBias - top * factor;

    // Two turns at a time, as the scores' registers alternate; two such in a row, so that places in the rings are constants.
    constexpr uint32_t kUnit = T::kUnitBytes;
    for (int u0 = 0; u0 < units; u0 += T::kRing) {
#pragma unroll
        for (int j = 0; j < T::kRing; ++j) {
            const int u = u0 + j;
            if (j == 2 && u >= units) break;
            const bool first = j % T::kBatch == 0, last = (j + 1) % T::kBatch == 0;
            const int set = j / 2 % kSets;
            if (first) {
                wait_batch();
                if constexpr (kMask != kMaskNone) {  // (their wait here: further on it would be one for the next copies)
                    mask[set][0].arrive();
                    mask[set][1].arrive();
                    if (kSets == 2) load_masks(mask[kSets - 1 - set], u + 3);
                }
            }
            const uint32_t ka = (j + 1) % T::kRing * kUnit, kn = (j + 2) % T::kRing * kUnit;
            const uint32_t va = (j + T::kRing - 1) % T::kRing * kUnit;
            if (j % 2 == 0) turn(u, s0, s1, p0, p1, ka, va, kn, mask[set][0], first, last);
            else turn(u, s1, s0, p1, p0, ka, va, kn, mask[set][1], first, last);
        }
    }
    // The last unit's values. The wait before its turn was one for them too where each turn has one; with two units a batch they
    // came with its own batch.
    if (T::kBatch > 1) wait_batch();
    {
        const uint32_t va = (units - 1) % T::kRing * kUnit;
        u32x4 vf[3];
        vf[0] = read_v(0, va);
        vf[1] = read_v(1, va);
#pragma unroll
        for (int n = 0; n < kSteps; ++n) {
            if (n + 2 < kSteps) vf[(n + 2) % 3] = read_v(n + 2, va);
            __builtin_amdgcn_sched_barrier(0);
            mfma_next<kBf16, T::kAccumulation, T::kAccumulation>(o[n % kBlocks], vf[n % 3], p1[n / kBlocks]);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    // the turns that other waves have more than this one: its share of their copies
    for (int u = units; u < wg_units; u += T::kBatch) {
        if (T::kBatch == 1) wait_batch();
        copy_batch(u);
        if (T::kBatch > 1) wait_batch();  // (the one that stood before turn u came before the last unit's values)
    }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) settle<T::kAccumulation>(o[b]);
    wait_vmcnt<0>();  // (no copy may be on its way when the workgroup's LDS goes to another)

    const int64_t out_row = static_cast<int64_t>(p.heads) * p.dim * 2;
    uint16_t* out = p.out + ((static_cast<int64_t>(job.b) * p.sq + job.q_start + row0) * p.heads + head) * p.dim;
    const auto ob = resource_of(out, (job.rows - row0 - 1) * out_row + p.dim * 2);
    const float sum = sum_halves(total);
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    // (the lane again: kept over the loop it would cost registers)
    const int place_of = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)), out_l32 = place_of % 32, out_half = place_of / 32;
    // element 4 g + j of block b is column 32 b + 8 g + 4 half + j: lanes 32 apart trade four columns, so that each
    // stores eight
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
            uint32_t h[2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    h[i][j] = pack2<kBf16>(o[b][(g + i) * 4 + j * 2] * inverse, o[b][(g + i) * 4 + j * 2 + 1] * inverse);
            const auto x = __builtin_amdgcn_permlane32_swap(h[0][0], h[1][0], false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(h[0][1], h[1][1], false, false);
            const int d = b * 32 + (g + out_half) * 8;
            __builtin_amdgcn_raw_buffer_store_b128(u32x4{x[0], y[0], x[1], y[1]}, ob,
                                                   d < p.dim ? static_cast<uint32_t>(out_l32 * out_row) + d * 2 : kPastEnd, 0, 0);
        }
}

template <int kDim, bool kBf16, int kMask>
int launch_attention_tiles(const AttnArgs& p, const AttnPlan& plan, hipStream_t stream) {
    const int64_t per_xcd = (plan.slots * p.heads + kNumXcd - 1) / kNumXcd;
    if (per_xcd * kNumXcd * 256 > 0xffffffffll) return FEATHER_ERR_UNSUPPORTED;
    AttnArgs args = p;
    args.by_slots = AttnDivisor::of(plan.slots);
    args.by_blocks = AttnDivisor::of((p.sq + 127) / 128);
    args.by_group = AttnDivisor::of(p.group);
    args.classes = 1;
    while (args.classes < kNumXcd && p.heads % (args.classes * 2) == 0) args.classes *= 2;
    args.class_heads = p.heads / args.classes;
    args.by_class = AttnDivisor::of(args.class_heads);
    auto* kernel = attention_tile_kernel<kDim, kBf16, kMask>;
    kernel<<<dim3(static_cast<uint32_t>(per_xcd * kNumXcd)), 256, 0, stream>>>(args, static_cast<int>(plan.slots), static_cast<int>(per_xcd));
    return hipGetLastError() == hipSuccess ? FEATHER_OK : FEATHER_ERR_LAUNCH;
}

}  // namespace feather
