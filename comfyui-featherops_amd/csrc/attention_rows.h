// Attention of few queries over many keys: decoded tokens, pooling queries, short prompts over a long cache.
//
// The keys and values are the work: they are read once, and a query's group of heads that share them
// are rows of one tile (row r is token r / group, head r % group). A workgroup has 32 rows and a run
// of keys; its four or eight waves take turns in tiles of 32 keys, each in LDS of its own, so that no
// wave waits for another before the end. There the waves' sums are joined through
// LDS, and where several workgroups share a row's keys, their sums through the workspace by the one
// that arrives last, in the order of the keys: the result does not depend on who that is.
//
// Bound by the memory's latency and rate: a wave has one tile of keys and one of values on their way, which makes 64 to
// 128 KB a CU. One token, 32 heads over 8, 32001 keys of 128: 31 us, 4.2 TB/s (a workgroup a block: 972); eight tokens over 1 to
// 4096 keys: 15 us of kernel, 3.1 TB/s. A join through the workspace costs 4 us and more, so that one query over 729 keys x 16 heads
// (7.8 us) is left to 16 workgroups.
#pragma once

#include "attention_device.h"

namespace feather {

template <int kDim>
struct AttnRows {
    static constexpr int kTileBytes = 32 * kDim * 2;
    static constexpr int kCopies = kTileBytes / 1024;
    static constexpr int kRing = 2 * kTileBytes;  // a wave's: keys and values
    // after the last tile: a wave's sums, 32 rows of kDim, the four values of a place swapped about against bank conflicts
    static_assert(32 * kDim * 4 <= kRing);
};

template <int kDim, bool kBf16, int kMask, int kWaves>
__global__ __launch_bounds__(64 * kWaves, kDim <= 128 ? 2 : 1) void attention_rows_kernel(const AttnArgs p, int slots, int total, int splits,
                                                                                      int least, uint32_t* counters, float* partials) {
    using T = AttnRows<kDim>;
    using Wave = AttnWave<kDim, kBf16, kMask, 1>;
    constexpr int kThreads = 64 * kWaves;
    __shared__ __attribute__((aligned(1024))) uint8_t rings[kWaves * T::kRing];
    __shared__ float tops[kWaves][32], totals[kWaves][32];

    // workgroup i runs on XCD i % 8: an XCD takes the row blocks that share keys
    const int per_xcd = static_cast<int>(gridDim.x / kNumXcd);
    const int id = static_cast<int>(blockIdx.x % kNumXcd) * per_xcd + static_cast<int>(blockIdx.x / kNumXcd);
    if (id >= total) return;
    const int rest = p.by_slots(id), slot = id - rest * slots;
    const int kv_head = p.by_splits(rest), split = rest - kv_head * splits;
    AttnJob job;
    if (!attn_job<32>(p, slot, p.group, job)) return;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int l32 = lane % 32, half = lane / 32;
    const int rows = min(32, job.rows - job.row0);
    // this lane's query, and the keys [0, limit) that it sees
    const int row = job.row0 + min(l32, rows - 1), token = p.by_group(row), head = kv_head * p.group + row - token * p.group;
    const int shift = job.keys - p.by_group(job.rows);
    const int limit = p.causal ? min(job.keys, token + shift + 1) : job.keys;
    const int seen = p.causal ? max(0, min(job.keys, p.by_group(job.row0 + rows - 1) + shift + 1)) : job.keys;
    const int every = p.causal ? min(job.keys, p.by_group(job.row0) + shift + 1) : job.keys;
    // the splits' runs of tiles: as even as whole tiles allow, none shorter than `least`
    const int all_tiles = (seen + 31) / 32;
    const int run = max(least, p.by_splits(all_tiles + splits - 1));
    const int live = max(1, (all_tiles + run - 1) / run);
    if (split >= live) return;
    const int first = split * run, tiles = min(run, all_tiles - first);

    const uint8_t* k = p.k + job.b * p.k_batch + job.k_start * p.k_row + kv_head * p.k_head;
    const uint8_t* v = p.v + job.b * p.v_batch + job.k_start * p.v_row + kv_head * p.v_head;
    const uint32_t ring = lds_addr_of(rings) + wave * T::kRing;
    uint32_t k_off[T::kCopies], v_off[T::kCopies];
#pragma unroll
    for (int i = 0; i < T::kCopies; ++i) {
        k_off[i] = tile_offset<kDim, false>(i, lane, p.k_row, p.dim);
        v_off[i] = tile_offset<kDim, true>(i, lane, p.v_row, p.dim);
    }
    auto copy = [&](const uint8_t* from, int64_t row_bytes, const uint32_t (&off)[T::kCopies], uint32_t at, int t) {
        const int64_t key0 = (first + t) * 32;
        const i32x4 buffer = buffer_of(from + key0 * row_bytes, (job.keys - key0 - 1) * row_bytes + p.dim * 2);
#pragma unroll
        for (int i = 0; i < T::kCopies; ++i) buffer_to_lds(buffer, off[i], at + i * 1024);
    };
    auto copy_k = [&](int t) { copy(k, p.k_row, k_off, ring, t); };
    auto copy_v = [&](int t) { copy(v, p.v_row, v_off, ring + T::kTileBytes, t); };
    Wave w;
    w.start(ring, ring + T::kTileBytes, p.scale);
    {
        const uint8_t* q = p.q + job.b * p.q_batch + (job.q_start + static_cast<int64_t>(token)) * p.q_row + head * p.q_head;
#pragma unroll
        for (int s = 0; s < Wave::kSteps; ++s) {
            const int d = s * 16 + half * 8;
            w.qf[s] = u32x4{};
            if (d < p.dim) __builtin_memcpy(&w.qf[s], q + d * 2, 16);
        }
    }
    if constexpr (kMask != kMaskNone)
        w.mask_row = p.mask + job.b * p.mask_batch + head * p.mask_head + token * p.mask_row;

    if (wave < tiles) {
        w.mask.load(w.mask_row, (first + wave) * 32, job.keys);
        copy_k(wave);
        copy_v(wave);
    }

    for (int t = wave; t < tiles; t += kWaves) {
        const int key0 = (first + t) * 32;
        const bool more = t + kWaves < tiles;
        f32x16 s[1];
        u32x4 pf[2];
        // The keys have landed (the values may be on their way); once read, the next tile's take their place, and likewise
        // the values.
        wait_vmcnt<T::kCopies>();
        asm volatile("" ::: "memory");
        w.scores(0, s);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if constexpr (kMask != kMaskNone) {
            // (a wait for the mask's values, which is one for the values as well: the next keys are copied behind it)
            wait_vmcnt<0>();
            w.masked(s, key0, limit, key0 + 32 > every);
            if (more) w.mask.load(w.mask_row, key0 + 32 * kWaves, job.keys);
        }
        if (more) copy_k(t + kWaves);
        if constexpr (kMask == kMaskNone) w.masked(s, key0, limit, key0 + 32 > every);
        w.weights(s, pf);
        if (more && kMask == kMaskNone) wait_vmcnt<T::kCopies>();
        else if (!more) wait_vmcnt<0>();
        asm volatile("" ::: "memory");
        w.add(0, pf);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) copy_v(t + kWaves);
    }

    // the waves' sums
    w.total = sum_halves(w.total);
    float* mine = reinterpret_cast<float*>(rings + wave * T::kRing);
    if (half == 0) {
        tops[wave][l32] = w.top;
        totals[wave][l32] = w.total;
    }
    if (l32 < rows) {
#pragma unroll
        for (int b = 0; b < Wave::kBlocks; ++b)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<float4*>(mine + l32 * kDim + ((b * 8 + g * 2 + half) ^ (l32 & 7)) * 4) =
                    make_float4(w.o[b][g * 4], w.o[b][g * 4 + 1], w.o[b][g * 4 + 2], w.o[b][g * 4 + 3]);
    }
    __syncthreads();

    const int quads = p.dim / 4;
    auto store = [&](int r, int c, f32x4 sum, float inverse) {
        const int tok = p.by_group(job.row0 + r), h = kv_head * p.group + job.row0 + r - tok * p.group;
        uint16_t* out = p.out + ((static_cast<int64_t>(job.b) * p.sq + job.q_start + tok) * p.heads + h) * p.dim + c * 4;
        *reinterpret_cast<uint2*>(out) =
            make_uint2(pack2<kBf16>(sum[0] * inverse, sum[1] * inverse), pack2<kBf16>(sum[2] * inverse, sum[3] * inverse));
    };
    // a row's sums, relative to the largest of the waves' maxima
    auto joined = [&](int r, int c, float& top, float& sum_of) {
        top = tops[0][r];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) top = fmaxf(top, tops[i][r]);
        f32x4 sum = f32x4{};
        sum_of = 0.0f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            const float by = __builtin_amdgcn_exp2f((tops[i][r] - top) * w.factor);
            sum_of += totals[i][r] * by;
            sum += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(rings + i * T::kRing) + r * kDim + (c ^ (r & 7)) * 4) * by;
        }
        return sum;
    };
    if (live == 1) {
        for (int u = threadIdx.x; u < rows * quads; u += kThreads) {
            const int r = p.by_quads(u), c = u - r * quads;
            float top, sum_of;
            const f32x4 sum = joined(r, c, top, sum_of);
            store(r, c, sum, sum_of == 0.0f ? 0.0f : 1.0f / sum_of);
        }
        return;
    }

    // Ordering: partials are written and read with agent-scope (sc1) accesses alone, which are coherent across
    // the XCDs. A store is acknowledged (vmcnt) once it is visible at agent scope; every wave waits for
    // that before the barrier that precedes the arrival count, and the last arrival's loads depend on
    // the count's answer.
    constexpr int kCoherent = 16;  // sc1
    constexpr int kRowFloats = kDim + 4, kPartBytes = 32 * kRowFloats * 4;  // top, total, two unused, the sums
    const int64_t place = (static_cast<int64_t>(kv_head) * slots + slot);
    const auto parts = resource_of(partials + place * splits * (kPartBytes / 4), static_cast<int64_t>(splits) * kPartBytes);
    for (int u = threadIdx.x; u < rows * quads; u += kThreads) {
        const int r = p.by_quads(u), c = u - r * quads;
        float top, sum_of;
        const f32x4 sum = joined(r, c, top, sum_of);
        const int at = split * kPartBytes + r * kRowFloats * 4;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum), parts, at + 16 + c * 16, 0, kCoherent);
        if (c == 0)
            __builtin_amdgcn_raw_buffer_store_b128(u32x4{f32_bits(top), f32_bits(sum_of), 0u, 0u}, parts, at, 0, kCoherent);
    }
    wait_vmcnt<0>();
    __shared__ int last;
    __syncthreads();
    if (threadIdx.x == 0)
        last = __hip_atomic_fetch_add(&counters[place], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<uint32_t>(live - 1);
    __syncthreads();
    if (!last) return;
    // Factors of the splits' sums, several threads a row; then the sums, several threads to a place if there are few rows.
    auto part = [&](int at) { return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(parts, at, 0, kCoherent)); };
    float* factors = reinterpret_cast<float*>(rings);  // [split][row]
    float* inverses = factors + kAttnMostSplits * 32;
    f32x4* sums = reinterpret_cast<f32x4*>(inverses + 32);
    {
        constexpr int kTeam = kThreads / 32, kEach = kAttnMostSplits / kTeam;
        const int r = threadIdx.x / kTeam, j = threadIdx.x % kTeam;
        f32x4 head_of[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (i * kTeam < live) head_of[i] = part(min(i * kTeam + j, live - 1) * kPartBytes + min(r, rows - 1) * kRowFloats * 4);
        float top = head_of[0][0];
#pragma unroll
        for (int i = 1; i < kEach; ++i)
            if (i * kTeam < live) top = fmaxf(top, head_of[i][0]);
#pragma unroll
        for (int m = 1; m < kTeam; m *= 2) top = fmaxf(top, __shfl_xor(top, m));
        float sum_of = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (i * kTeam + j >= live) continue;
            const float by = __builtin_amdgcn_exp2f((head_of[i][0] - top) * w.factor);
            factors[(i * kTeam + j) * 32 + r] = by;
            sum_of += head_of[i][1] * by;
        }
#pragma unroll
        for (int m = 1; m < kTeam; m *= 2) sum_of += __shfl_xor(sum_of, m);
        if (j == 0) inverses[r] = sum_of == 0.0f ? 0.0f : 1.0f / sum_of;
    }
    __syncthreads();
    const int places = rows * quads;
    int teams = 1;
    while (teams * 2 * places <= kThreads) teams *= 2;
    auto gather = [&](int u, int from) {
        const int r = p.by_quads(u), at = r * kRowFloats * 4 + 16 + (u - r * quads) * 16;
        f32x4 sum = f32x4{};
        constexpr int kAhead = 8;
        for (int s0 = from; s0 < live; s0 += kAhead * teams) {
            f32x4 values[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (s0 + i * teams < live) values[i] = part((s0 + i * teams) * kPartBytes + at);
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (s0 + i * teams < live) sum += values[i] * factors[(s0 + i * teams) * 32 + r];
        }
        return sum;
    };
    if (teams == 1) {
        for (int u = threadIdx.x; u < places; u += kThreads) {
            const int r = p.by_quads(u);
            store(r, u - r * quads, gather(u, 0), inverses[r]);
        }
    } else {
        const int team = threadIdx.x / places, u = threadIdx.x - team * places;
        if (team < teams) sums[team * places + u] = gather(u, team);
        __syncthreads();
        if (team == 0) {
            f32x4 sum = sums[u];
            for (int i = 1; i < teams; ++i) sum += sums[i * places + u];
            const int r = p.by_quads(u);
            store(r, u - r * quads, sum, inverses[r]);
        }
    }
    if (threadIdx.x == 0)  // ready for the next call on this stream
        __hip_atomic_store(&counters[place], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int kDim, bool kBf16, int kMask, int kWaves>
int launch_attention_rows(const AttnArgs& p, const AttnPlan& plan, void* workspace, hipStream_t stream) {
    const int64_t total = plan.slots * p.kv_heads * plan.splits;
    const int64_t grid = (total + kNumXcd - 1) / kNumXcd * kNumXcd;
    if (grid * 64 * kWaves > 0xffffffffll) return FEATHER_ERR_UNSUPPORTED;
    AttnArgs args = p;
    args.by_slots = AttnDivisor::of(plan.slots);
    args.by_blocks = AttnDivisor::of((static_cast<int64_t>(p.sq) * p.group + 31) / 32);
    args.by_group = AttnDivisor::of(p.group);
    args.by_splits = AttnDivisor::of(plan.splits);
    args.by_quads = AttnDivisor::of(p.dim / 4);
    auto* kernel = attention_rows_kernel<kDim, kBf16, kMask, kWaves>;
    kernel<<<dim3(static_cast<uint32_t>(grid)), 64 * kWaves, 0, stream>>>(
        args, static_cast<int>(plan.slots), static_cast<int>(total), plan.splits, plan.least, static_cast<uint32_t*>(workspace),
        reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kAttnCounterBytes));
    return hipGetLastError() == hipSuccess ? FEATHER_OK : FEATHER_ERR_LAUNCH;
}

}  // namespace feather
