#include "kernels/prefix_plan.h"

#include <algorithm>
#include <string>

#include "util/error.h"

namespace illm {
namespace ops {

// Rows (members times G) of a tile: wide, or narrow.  Narrow tiles of eight rows leave a block half the registers of sixteen, so that twice as many share an SM, and are
// taken while they hold two members (16 sequences of 32 / 32 heads behind 2,048 positions 17.0 us and 23.2; of 32 / 8 heads 13.9 and 17.1).
static constexpr int kFewRows = 8, kNarrowRows = 16, kWideRows = 256;
// Wide tiles where a group takes more narrow ones than this: 32 / 32 heads behind 8,192 positions, 32 sequences 52 us narrow and 54 wide, 48 sequences 71 and 59, 128
// sequences 180 and 86; 32 / 8 heads, 8 sequences 20 and 19, 16 sequences 30 and 24; behind 512 positions the two are nearly alike.
static constexpr int kNarrowMost = 4;

PrefixPlanSizes prefix_plan_sizes(const std::vector<PrefixGroup>& groups, const int* lens, int T, int G) {
    if (T < 1 || T > 65535) throw KernelError("a plan of common prefixes takes 1 to 65535 tokens, found " + std::to_string(T));
    if (G < 1 || G > kNarrowRows) throw KernelError("a plan of common prefixes takes 1 to 16 query heads per key/value head, found " + std::to_string(G));
    PrefixPlanSizes s;
    s.T = T;
    std::vector<int> start((size_t)T, 0);
    int most = 0;               // members of a group
    for (const PrefixGroup& g : groups) {
        if (g.members.empty()) throw KernelError("a group of tokens with a common prefix needs at least one token");
        if (g.prefix < 1) throw KernelError("a common prefix must have at least one position, found " + std::to_string(g.prefix));
        for (int t : g.members) {
            if (t < 0 || t >= T) throw KernelError("token " + std::to_string(t) + " of a group is outside the step's " + std::to_string(T));
            if (start[(size_t)t]) throw KernelError("token " + std::to_string(t) + " is in two groups (or twice in one)");
            if (lens[t] < g.prefix)
                throw KernelError("token " + std::to_string(t) + " sees " + std::to_string(lens[t]) + " positions, fewer than the common prefix of " + std::to_string(g.prefix));
            start[(size_t)t] = g.prefix;
        }
        most = std::max(most, (int)g.members.size());
        s.longest_prefix = std::max(s.longest_prefix, g.prefix);
    }
    const int narrow = (2 * G <= kFewRows ? kFewRows : kNarrowRows) / G;
    s.wide = most > kNarrowMost * narrow;
    s.per_tile = s.wide ? kWideRows / G : narrow;
    for (const PrefixGroup& g : groups) s.tiles += ((int)g.members.size() + s.per_tile - 1) / s.per_tile;
    for (int t = 0; t < T; t++) {
        if (lens[t] < 1) throw KernelError("token " + std::to_string(t) + " sees no position");
        s.longest_rest = std::max(s.longest_rest, lens[t] - start[(size_t)t]);
    }
    return s;
}

bool shared_prefix_pays(long long saved_rows, long long sequences, bool int8) {
    return saved_rows >= std::min<long long>(int8 ? 32768 + 8192 * sequences : 131072 + 12288 * sequences, 393216);
}

void prefix_plan_fill(const std::vector<PrefixGroup>& groups, const PrefixPlanSizes& s, int* out) {
    std::fill(out, out + s.ints(), 0);
    int tile = 0;
    const int per = s.per_tile;
    for (const PrefixGroup& g : groups)
        for (size_t i = 0; i < g.members.size(); i += (size_t)per) {
            const int n = std::min(per, (int)(g.members.size() - i));
            out[4 * tile] = n;
            out[4 * tile + 1] = g.prefix;
            for (int k = 0; k < n; k++) {
                out[s.members_at() + tile * per + k] = g.members[i + (size_t)k];
                out[s.start_at() + g.members[i + (size_t)k]] = g.prefix;
            }
            tile++;
        }
}

}  // namespace ops
}  // namespace illm
