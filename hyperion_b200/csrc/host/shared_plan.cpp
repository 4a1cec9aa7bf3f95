#include "shared_plan.hpp"

#include <algorithm>
#include <string>

#include "cache_index.hpp"

namespace hb {
namespace {

constexpr int64_t TILE_ROWS = 256;       // (token, head) rows of an item of the tile kernel
constexpr int64_t MOST_STRIP_ROWS = 64;  // of a range that the strip kernel serves, eight or sixteen rows an item
constexpr int64_t WHOLE_STRIP = 4;       // tiles of a strip that stays uncut where there is a block for each
constexpr int64_t MOST_TOGETHER = 8;     // blocks of a cluster
constexpr int64_t WHOLE_TOGETHER = 2;    // tiles of a run that a cluster is not made for
constexpr int64_t SAVED_TILES = 3;       // how many tiles of a strip the joining by a kernel of its own takes as long as
constexpr int64_t KEYS = 128;            // keys of a tile, in which shares are counted

// A range of keys that every one of a run of tokens sees (but for the last of them, which the tokens' own positions bound).
struct Run {
    int64_t token, count, row, low, high;
    bool own;
    int64_t operand = 0;  // of the range's first tile
};

int64_t tiles_of(const Run& run) { return (run.high + KEYS - 1) / KEYS - run.low / KEYS; }

// Cuts the runs, one behind the other, into as many walks of equal cost as there are blocks.  An item costs `overhead` tiles beside its own (its queries' way in, its
// rows' way out) and has `least` tiles at least; runs of up to `whole` tiles stay uncut where there is a block for each.
Walk cut(const std::vector<Run>& runs, int64_t blocks, double overhead, int64_t least, int64_t whole) {
    Walk walk;
    walk.first.push_back(0);
    if (runs.empty()) return walk;
    int64_t left = 0, longest = 0, runs_left = (int64_t)runs.size();  // tiles and runs that are yet to be given out
    for (const Run& run : runs) {
        left += tiles_of(run);
        longest = std::max(longest, tiles_of(run));
    }
    const bool uncut = longest <= whole && (int64_t)runs.size() <= blocks;
    double budget = 0, used = 0;
    const auto open_block = [&] {  // with an equal share of what is left
        const double blocks_left = (double)std::max<int64_t>(1, blocks - walk.blocks());
        budget = uncut ? overhead + (double)longest : std::max(((double)left + overhead * ((double)runs_left + blocks_left - 1)) / blocks_left, overhead + (double)least);
        used = 0;
    };
    const auto next_block = [&] {
        walk.first.push_back((int)(walk.items.size() / ITEM_WORDS));
        open_block();
    };
    open_block();
    for (const Run& run : runs) {
        const int64_t base = run.low / KEYS, tiles = tiles_of(run);
        int64_t done = 0;
        for (int piece = 0; done < tiles; ++piece) {
            int64_t take = tiles - done;
            if (walk.blocks() + 1 < blocks) {  // the last block takes what is left
                const int64_t room = (int64_t)(budget - used - overhead + 0.5);
                if (used > 0 && room < std::min(least, take)) {
                    next_block();
                    --piece;
                    continue;
                }
                if (take - room >= least) take = std::max(room, least);  // what would be left over must be worth an item
            }
            const int64_t low = std::max(run.low, (base + done) * KEYS), high = std::min(run.high, (base + done + take) * KEYS);
            for (int64_t word : {run.token, run.count, run.row, low, high, (int64_t)piece + (run.own ? OWN_PIECE : 0), run.operand + done}) walk.items.push_back((int)word);
            used += overhead + (double)take;
            done += take;
            left -= take;
        }
        --runs_left;
    }
    next_block();
    return walk;
}

void require(bool condition, const char* message) {
    if (!condition) throw Failure{BAD_ARGUMENT, message};
}

}  // namespace

SharedPlan plan_shared(const std::vector<int64_t>& counts, const std::vector<int64_t>& lengths, const std::vector<SharedGroup>& groups, int64_t heads, int64_t kv_heads, int64_t sms) {
    require(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "plan_shared: query heads do not divide over key/value heads");
    require(sms > 0, "plan_shared: a device has multiprocessors");
    const int64_t requests = (int64_t)counts.size(), group = heads / kv_heads, most = (int64_t(1) << 31) - 1 - KEYS;
    std::vector<int64_t> start(requests + 1, 0), own_from(requests, 0);
    SharedPlan plan;
    for (int64_t r = 0; r < requests; ++r) {
        require(counts[r] >= 0 && lengths[r] >= 0, "plan_shared: a count of queries and a length for each request, none of them negative");
        require(counts[r] <= most && lengths[r] <= most, "plan_shared: counts and positions fit 32 bits");
        start[r + 1] = start[r] + counts[r];
        require(start[r + 1] <= most, "plan_shared: the tokens of a step fit 32 bits");
        if (counts[r]) plan.longest = std::max(plan.longest, lengths[r]);
    }
    const int64_t tokens = start[requests];
    std::vector<Run> ranges;
    int64_t after = 0;
    for (const SharedGroup& g : groups) {
        require(g.first >= after && g.members >= 0 && g.members <= requests && g.first <= requests - g.members && g.positions >= 0, "plan_shared: groups of consecutive requests, in order, that do not overlap");
        after = g.first + g.members;
        int64_t row = -1;  // of a request that is in the step
        for (int64_t r = g.first; r < after; ++r) {
            if (!counts[r]) continue;
            require(lengths[r] - counts[r] >= g.positions || !g.positions, "plan_shared: every query of a group sees all of its shared positions");
            own_from[r] = g.positions;
            if (row < 0) row = r;
        }
        if (row >= 0 && g.positions) ranges.push_back({start[g.first], start[after] - start[g.first], row, 0, g.positions, false});
    }
    for (int64_t r = 0; r < requests; ++r)
        if (counts[r] && lengths[r] > own_from[r]) ranges.push_back({start[r], counts[r], r, own_from[r], lengths[r], true});

    const auto is_wide = [&](const Run& range) { return range.count * group > MOST_STRIP_ROWS; };
    for (const Run& range : ranges)
        if (!is_wide(range) && range.count * group > 8) plan.strip_rows = 16;
    int64_t distinct = 0;
    for (Run& range : ranges) {
        if (!is_wide(range)) continue;
        range.operand = distinct;
        distinct += tiles_of(range);
        require(distinct <= most / 4, "plan_shared: the tiles of a step fit 32 bits");
        for (int64_t at = range.low / KEYS * KEYS; at < range.high; at += KEYS)
            for (int64_t word : {range.row, at, range.low, range.high}) plan.operands.push_back((int)word);
    }
    const auto runs_of = [&](bool wide, int64_t rows) {
        const int64_t per = std::max<int64_t>(1, rows / group);
        std::vector<Run> runs;
        for (const Run& range : ranges)
            if (is_wide(range) == wide)
                for (int64_t at = 0; at < range.count; at += per)
                    runs.push_back({range.token + at, std::min(per, range.count - at), range.row, range.low, range.high, range.own, range.operand});
        return runs;
    };
    const std::vector<Run> strips = runs_of(false, plan.strip_rows), tiles = runs_of(true, TILE_ROWS);
    const int64_t strips_across = kv_heads * ((group + plan.strip_rows - 1) / plan.strip_rows), tiles_across = kv_heads * ((group + TILE_ROWS - 1) / TILE_ROWS);
    // Where a step has both kinds they run side by side, each on a part of the device that its work asks for.  A tile of 256 rows takes an SM some 2.1 us and an item of them 4
    // besides, a tile of a strip 0.65 (three blocks share the SM) and a strip 1.3.
    int64_t tile_sms = tiles.empty() ? 0 : sms;
    if (!tiles.empty() && !strips.empty()) {
        double tile_work = 0, strip_work = 0;
        for (const Run& run : tiles) tile_work += (2.1 * (double)tiles_of(run) + 4) * (double)tiles_across;
        for (const Run& run : strips) strip_work += (0.65 * (double)tiles_of(run) + 1.3) * (double)strips_across;
        tile_sms = std::max<int64_t>(1, std::min<int64_t>(sms - 1, (int64_t)((double)sms * tile_work / (tile_work + strip_work) + 0.5)));
        tile_sms = std::min(sms, std::max<int64_t>(1, (tile_sms + tiles_across / 2) / tiles_across) * tiles_across);
    }
    const int64_t strip_sms = tile_sms < sms ? sms - tile_sms : sms;  // what is left, or all of it one after the other
    // Steps of strips alone in which every token has one run: a run's shares go to up to eight blocks that stand together and join them (a cluster), without a kernel behind, as
    // long as the longest run's shares are not much longer than shares over the whole device would be (one request at 5,120 positions, five tiles a block: 11.8 us against 10.2 with the
    // joining, and a kernel less; at 7,000, seven: 14.0 against 12.0, and from there on the whole device is used).  Runs of up to two tiles stay whole: 5.4 us against 6.1.
    const int64_t slots = strip_sms * (plan.strip_rows == 8 ? 3 : 2) / strips_across;
    int64_t with_own = 0;
    for (const Run& range : ranges) with_own += range.own ? range.count : 0;
    if (tiles.empty() && !strips.empty() && with_own == (int64_t)tokens && std::all_of(ranges.begin(), ranges.end(), [](const Run& range) { return range.own; })) {
        int64_t longest = 0, total = 0;
        for (const Run& run : strips) longest = std::max(longest, tiles_of(run)), total += tiles_of(run);
        const int64_t blocks = std::min({MOST_TOGETHER, slots / (int64_t)strips.size(), longest});
        const int64_t share = blocks > 1 ? (longest + blocks - 1) / blocks : 0, spread = std::max<int64_t>(2, (total + slots - 1) / std::max<int64_t>(1, slots));
        if (longest > WHOLE_TOGETHER && blocks > 1 && share <= spread + SAVED_TILES) plan.together = (int)blocks;
    }
    if (plan.together) {
        plan.strips.first.push_back(0);
        for (const Run& run : strips) {
            const int64_t first = run.low / KEYS, n = tiles_of(run);
            for (int64_t i = 0; i < plan.together; ++i) {
                const int64_t from = first + n * i / plan.together, to = first + n * (i + 1) / plan.together;
                const bool empty = from == to;
                for (int64_t word : {run.token, run.count, run.row, empty ? 0 : std::max(run.low, from * KEYS), empty ? 0 : std::min(run.high, to * KEYS), i + OWN_PIECE, run.operand})
                    plan.strips.items.push_back((int)word);
                plan.strips.first.push_back((int)plan.strips.first.size());
            }
        }
    } else {
        plan.strips = cut(strips, std::max<int64_t>(1, slots), 0.75, 2, WHOLE_STRIP);
    }
    plan.tiles = cut(tiles, std::max<int64_t>(1, tile_sms / tiles_across), 1.5, 2, 2);

    std::vector<int> of_group(tokens, 0), of_own(tokens, 0);
    for (const Walk* walk : {&plan.strips, &plan.tiles})
        for (size_t i = 0; i < walk->items.size(); i += ITEM_WORDS)
            for (int t = walk->items[i]; t < walk->items[i] + walk->items[i + 1]; ++t) ++(walk->items[i + 5] & OWN_PIECE ? of_own : of_group)[t];
    plan.starts.assign(tokens + 1, 0);
    plan.own.assign(tokens, 0);
    plan.last.assign(tokens, 0);
    for (int64_t r = 0; r < requests; ++r)
        for (int64_t i = 0; i < counts[r]; ++i) plan.last[start[r] + i] = (int)std::max<int64_t>(-1, lengths[r] - counts[r] + i);
    int64_t pieces = 0;
    for (int64_t t = 0; t < tokens; ++t) {
        plan.starts[t] = (int)pieces;
        plan.own[t] = (int)(pieces + of_group[t]);
        pieces += of_group[t] + of_own[t];
        plan.joined |= of_group[t] + of_own[t] != 1;
        require(pieces <= most, "plan_shared: the pieces of a step fit 32 bits");
    }
    plan.starts[tokens] = (int)pieces;
    return plan;
}

}  // namespace hb
