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
// Whether a decode step of `sequences` sequences should walk common prefixes once, in an entry of eight-bit (int8) or bfloat16 rows.  saved_rows: the rows (positions times
// kv heads) that it would not have to read again, a prefix counted once for every sequence of its group but one.
//   bfloat16: 131,072 rows and 12,288 more per sequence, eight bits: 32,768 and 8,192, both at most 393,216.
// Measured in the engine, a layer's time walked once less its time sequence by sequence, us, 100 positions behind the prefix; heads 32 / 8 of 128 unless others are named,
// thousands of rows saved in front:
//   bfloat16 (against the kernel that rotates, writes and attends in one): 4 sequences 96: +2.8, 192: -3.1 (32 / 32 heads 96: +2.7, 192: -1.3; heads of 64 96: +1.7, 192: -2.4);
//   8: 112: +1.9, 224: -2.8 (32 / 32 heads 224: +2.0, 448: -8.4); 16: 240: +3.9, 480: -5.8; 32: 248: +3.6, 496: -6.2; 64: 252: +2.8, 504: -8.0.
//   Eight bits: 2: 32: +3.9, 64: -2.2; 4: 24: -2.9, 96: -1.5; 8: 56: -3.6; 16: 120: -0.7, 240: +3.0, 480: -4.1; 32: 248: -4.8; 64: 504: -9.3.  There the other side is cut by
//   the cache's longest sequence (16,384 here), which costs it some us; with a limit at the sequences' lengths 16 sequences 120: +1.2, 240: -2.2; 64: 252: +7.3, 504: -1.6.
bool shared_prefix_pays(long long saved_rows, long long sequences, bool int8);
// Fills out[0 .. sizes.ints()); sizes.tiles may be larger than the plan needs (the rest are empty tiles).
void prefix_plan_fill(const std::vector<PrefixGroup>& groups, const PrefixPlanSizes& sizes, int* out);

}  // namespace ops
}  // namespace illm
