// The plan of a step of attention behind shared positions (csrc/attention_shared*.cu): which block of which kernel walks which keys for which tokens.
#pragma once
#include <cstdint>
#include <vector>

namespace hb {

struct SharedGroup {
    int64_t first, members, positions;  // requests first .. first + members - 1 hold the same pages for their first `positions` positions
};

// An item: first token, tokens, table row, first key, last key + 1, piece, operand tile.  `piece` is the item's number among the shares of its range; a token's pieces are those of
// its group's positions, from starts[token] on, and those of its own request's, from own[token] on: an item of the latter kind has OWN_PIECE added.  `operand tile`: where the item's
// first tile stands among the plan's operands.
constexpr int ITEM_WORDS = 7;
constexpr int OWN_PIECE = 1 << 30;

struct Walk {  // of one kernel: block b takes items first[b] .. first[b + 1] - 1
    std::vector<int> items, first;
    int blocks() const { return (int)first.size() - 1; }
};

struct SharedPlan {
    Walk strips, tiles;
    int strip_rows = 8;
    // 0, or how many blocks in a row walk one run between them, an item each (an empty one is keys 0 to 0), and put its pieces together themselves: a cluster.
    int together = 0;
    // The tiles of the wide ranges, each as (table row, first position, first key, last key + 1 of its range): what 8-bit records are made into operands for.
    std::vector<int> operands;
    std::vector<int> last, starts, own;  // the last position a token sees, its first piece, its first piece of its own request's positions
    bool joined = false;                 // some token has another number of pieces than one
    int64_t longest = 0;
};

SharedPlan plan_shared(const std::vector<int64_t>& counts, const std::vector<int64_t>& lengths, const std::vector<SharedGroup>& groups, int64_t heads, int64_t kv_heads, int64_t sms);

}  // namespace hb
