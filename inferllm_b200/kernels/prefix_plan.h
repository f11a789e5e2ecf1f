// The plan of a step's tokens whose sequences hold their first positions in common (csrc/attention_pages.cu, attention_tiles.cu), made on the
// host once per step: which tokens walk which positions together.
#pragma once
#include <vector>

namespace illm {
namespace ops {

// Tokens that see the same first `prefix` positions, held by the same pages.
struct PrefixGroup {
    int prefix = 0;
    std::vector<int> members;
};

struct PrefixPlanSizes {
    int T = 0;                  // tokens of the step
    int tiles = 0;              // groups in pieces that fit the rows of a block's products
    bool wide = false;          // pieces of 256 rows (attention_tiles.cu) or of 8 or 16 (attention_pages.cu)
    int longest_prefix = 0;     // positions
    int longest_rest = 0;       // the most positions that a token has for itself
    int per_tile = 0;           // members that fit a tile
    int ints() const { return members_at() + (tiles * per_tile + 3) / 4 * 4; }
    // where its arrays begin: tiles [tiles][4], start [T], members [tiles][per_tile]
    int start_at() const { return 4 * tiles; }
    int members_at() const { return 4 * tiles + (T + 3) / 4 * 4; }
};

// lens[t]: the positions that token t sees; G: query heads per key/value head, at most 16.  KernelError for a token outside the step or in
// two groups, an empty group, a prefix that is not positive or longer than a member sees.
PrefixPlanSizes prefix_plan_sizes(const std::vector<PrefixGroup>& groups, const int* lens, int T, int G);
// Fills out[0 .. sizes.ints()); sizes.tiles may be larger than the plan needs (the rest are empty tiles).
void prefix_plan_fill(const std::vector<PrefixGroup>& groups, const PrefixPlanSizes& sizes, int* out);

}  // namespace ops
}  // namespace illm
