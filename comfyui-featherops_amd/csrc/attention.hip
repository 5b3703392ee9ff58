// Which attention kernel takes a call.
//
// Three forms: attention_tiles.h (128 queries of a head a workgroup), and attention_rows.h with 4 or 8 waves and the keys
// of 32 rows shared by up to 64 workgroups. Each has a time, in microseconds, of a fixed part, a part for each
// workgroup that a CU gets, and one for its tiles: by their latency one after the other where a CU has one workgroup,
// by throughput where it has several. The constants were fitted to samples without lengths, before masks were read by words and blocks
// dealt out among the XCDs. With the kernels as they are, over 26,690 shapes (1 to 8 samples with and without lengths, 2 to 30 packed
// sequences, 1 to 40 heads in groups of 1 to 8, 1 to 16384 queries and keys, a third causal, a fifth with masks), each form and
// split timed on an MI355X: the form taken is 1.6% slower than the fastest of all in the mean, 10% at the 95th percentile; with lengths,
// which the host does not know, 2.3% and 13%, packed 1.8% and 12%. Most often fastest: few rows with 4 waves and unshared
// keys (43% of the shapes), with 8 (15%), blocks of 128 queries (25%), shared keys (18%).
#include "attention.h"

#include <algorithm>

namespace feather {
namespace {

struct Times {
    double call, workgroup, latency, throughput;  // the last two for 32 keys
};
struct DimTimes {
    int dim;
    Times tiles, masked_tiles, rows[2];  // rows: of 4 and 8 waves (a wide head has no 8)
};
constexpr DimTimes kTimes[] = {
    {64, {3.67, 1.74, 0.376, 0.304}, {4.23, 2.96, 0.667, 0.423}, {{3.48, 1.14, 0.807, 0.447}, {2.78, 2.05, 0.973, 0.804}}},
    {96, {3.24, 2.74, 0.430, 0.381}, {2.92, 4.77, 0.736, 0.534}, {{3.32, 1.67, 0.955, 0.666}, {0.45, 4.53, 1.312, 1.312}}},
    {128, {3.65, 2.97, 0.477, 0.477}, {2.70, 5.41, 0.801, 0.591}, {{2.73, 2.67, 1.082, 0.816}, {0.47, 5.34, 1.465, 1.465}}},
    {256, {6.80, 2.77, 0.933, 0.933}, {7.72, 3.97, 1.374, 1.374}, {{0.54, 7.63, 1.821, 1.821}, {}}},
};
// joining the sums of several workgroups: a call, and each row of each of them (half of that with 8 waves)
constexpr double kJoin = 3.8, kJoinRow = 0.00012;  // the latter times the head's dimension
constexpr int kCus = 256;
constexpr int kLeastTiles = 4;  // a split's, fewer do not pay for its join

int64_t parts(int64_t n, int64_t of) { return (n + of - 1) / of; }

double time_of(const Times& t, int64_t workgroups, double most, double mean) {
    const double each = static_cast<double>(parts(workgroups, kCus));
    return t.call + t.workgroup * each + std::max(t.latency * most, t.throughput * mean * each);
}

}  // namespace

AttnPlan attention_plan(const AttnArgs& p) {
    const bool packed = p.q_offsets;
    // Queries and keys of a sample. Of packed sequences the host knows the sums alone: as if they were alike, the longest twice
    // the mean.
    const int64_t queries = packed ? parts(p.sq, p.batch) : p.sq, keys = packed ? parts(p.sk, p.batch) : p.sk;
    const int64_t longest = packed ? std::min<int64_t>(p.sk, 2 * keys) : keys;
    auto slots = [&](int64_t per_token, int64_t block) {
        return packed ? p.sq * per_token / block + p.batch + 2 : p.batch * parts(p.sq * per_token, block);
    };
    // the part of the keys that a query sees in the mean
    double seen = 1.0;
    if (p.causal && keys > 0) {
        const double n = static_cast<double>(queries), m = static_cast<double>(keys);
        seen = m >= n ? 1.0 - (n - 1.0) / (2.0 * m) : (m + 1.0) / (2.0 * n);
    }
    const DimTimes* times = kTimes;
    while (times->dim < p.dim) ++times;

    AttnPlan best{};
    best.slots = slots(1, 128);
    best.splits = 1;
    best.least = kLeastTiles;
    double least = time_of(p.mask_type ? times->masked_tiles : times->tiles, p.batch * parts(queries, 128) * p.heads,
                           static_cast<double>(longest) / 32.0 + 1.0, seen * static_cast<double>(keys) / 32.0 + 1.0);
    const int64_t row_slots = slots(p.group, 32), places = row_slots * p.kv_heads;
    const int64_t jobs = p.batch * parts(queries * p.group, 32) * p.kv_heads, tiles = std::max<int64_t>(1, parts(longest, 32));
    const double rows = static_cast<double>(std::min<int64_t>(queries * p.group, 32));
    for (int form = 0; form < (times->dim == 256 ? 1 : 2); ++form) {
        const int waves = form ? 8 : 4;
        for (int splits = 1; splits <= kAttnMostSplits; splits *= 2) {
            const int64_t run = std::max<int64_t>(kLeastTiles, parts(tiles, splits)), live = parts(tiles, run);
            if (splits > 1 && (live <= splits / 2 || places > static_cast<int64_t>(kAttnCounterBytes / 4))) break;
            const double most = static_cast<double>(parts(std::min(run, tiles), waves));
            double time = time_of(times->rows[form], jobs * live, most, std::max(1.0, most * seen * static_cast<double>(keys) / longest));
            if (live > 1) time += kJoin + kJoinRow * times->dim * (form ? 0.55 : 1.0) * rows * static_cast<double>(live);
            if (time >= least) continue;
            least = time;
            best.waves = waves;
            best.slots = row_slots;
            best.splits = static_cast<int>(live);
        }
    }
    if (best.waves && best.splits > 1)
        best.workspace = kAttnCounterBytes + static_cast<size_t>(places) * best.splits * 32 * (times->dim + 4) * 4;
    return best;
}

}  // namespace feather
