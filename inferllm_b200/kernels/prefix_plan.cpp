#include "kernels/prefix_plan.h"

#include <algorithm>
#include <string>

#include "util/error.h"

namespace illm {
namespace ops {

// Rows (members times G) of a tile, and up to which group the first of them are taken.
static constexpr int kFewRows = 8, kFewMost = 8, kNarrowRows = 16, kWideRows = 256;
// Narrow tiles times key/value heads from which on wide ones are taken where a group has more rows than a narrow one.
static constexpr int kNarrowMost = 24;

PrefixPlanSizes prefix_plan_sizes(const std::vector<PrefixGroup>& groups, const int* lens, int T, int G, int kv_heads) {
    if (T < 1 || T > 65535) throw KernelError("a plan of common prefixes takes 1 to 65535 tokens, found " + std::to_string(T));
    if (G < 1 || G > kNarrowRows) throw KernelError("a plan of common prefixes takes 1 to 16 query heads per key/value head, found " + std::to_string(G));
    if (kv_heads < 1) throw KernelError("a plan of common prefixes needs at least one key/value head, found " + std::to_string(kv_heads));
    PrefixPlanSizes s;
    s.T = T;
    std::vector<int> start((size_t)T, 0);
    int rows = 0;
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
        rows = std::max(rows, (int)g.members.size() * G);
        s.longest_prefix = std::max(s.longest_prefix, g.prefix);
    }
    auto tiles_of = [&](int per) {
        int n = 0;
        for (const PrefixGroup& g : groups) n += ((int)g.members.size() + per - 1) / per;
        return n;
    };
    s.wide = rows > kNarrowRows && (long long)tiles_of(kNarrowRows / G) * kv_heads >= kNarrowMost;
    s.per_tile = (s.wide ? kWideRows : rows <= kFewMost && G <= kFewRows ? kFewRows : kNarrowRows) / G;
    s.tiles = tiles_of(s.per_tile);
    for (int t = 0; t < T; t++) {
        if (lens[t] < 1) throw KernelError("token " + std::to_string(t) + " sees no position");
        s.longest_rest = std::max(s.longest_rest, lens[t] - start[(size_t)t]);
    }
    return s;
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
