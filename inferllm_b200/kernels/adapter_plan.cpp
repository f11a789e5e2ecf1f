#include "kernels/adapter_plan.h"

#include <algorithm>
#include <string>

#include "util/error.h"

namespace illm {
namespace ops {

static int groups_of(int rank) { return (rank + ADAPTER_GROUP - 1) / ADAPTER_GROUP; }

static std::vector<int> named(const int* index, int from, int to) {
    std::vector<int> out(index + from, index + to);
    std::sort(out.begin(), out.end());
    out.erase(std::unique(out.begin(), out.end()), out.end());
    if (!out.empty() && out.front() < 0) out.erase(out.begin());
    return out;
}
static int tile_end(int t0, int T) { return std::min(T, t0 + ADAPTER_TILE); }

AdapterPlanSizes adapter_plan_sizes(const int* index, int T, const int* ranks, int count) {
    if (T < 0 || T > 524280) throw KernelError("adapters: a step of " + std::to_string(T) + " tokens is outside [0, 524280]");
    for (int a = 0; a < count; a++)
        if (ranks[a] < 0 || ranks[a] > ADAPTER_GROUP * ADAPTER_MAX_GROUPS)
            throw KernelError("adapters: adapter " + std::to_string(a) + " has rank " + std::to_string(ranks[a]) + ", outside [0, 256]");
    for (int t = 0; t < T; t++)
        if (index[t] < -1 || index[t] >= count)
            throw KernelError("adapters: token " + std::to_string(t) + " names adapter " + std::to_string(index[t]) + " of " + std::to_string(count));
    AdapterPlanSizes s{T, 0, 0, 0};
    for (int a : named(index, 0, T)) {
        s.slots++;
        s.groups += groups_of(ranks[a]);
    }
    if (adapter_tiled(T, s.slots))
        for (int t0 = 0; t0 < T; t0 += ADAPTER_TILE) {
            int g = 0;
            for (int a : named(index, t0, tile_end(t0, T))) g += groups_of(ranks[a]);
            s.chunks += (g + ADAPTER_CHUNK - 1) / ADAPTER_CHUNK;
        }
    return s;
}

AdapterPlanSizes adapter_plan_bound(int T, int count, int max_rank, bool one_sequence) {
    const int slots = one_sequence ? std::min(1, T) : std::min(T, count);
    AdapterPlanSizes s{T, slots, slots * groups_of(max_rank), 0};
    if (adapter_tiled(T, slots))
        for (int t0 = 0; t0 < T; t0 += ADAPTER_TILE) {
            const int adapters = std::min(tile_end(t0, T) - t0, slots);
            s.chunks += (adapters * groups_of(max_rank) + ADAPTER_CHUNK - 1) / ADAPTER_CHUNK;
        }
    return s;
}

void adapter_plan_fill(const int* index, int T, const int* ranks, int count, const AdapterPlanSizes& sizes, int* out) {
    const AdapterPlanSizes least = adapter_plan_sizes(index, T, ranks, count);
    const bool tiled = adapter_tiled(T, sizes.slots);       // (room for more adapters than there are may mean rows)
    if (sizes.T != T || sizes.slots < least.slots || sizes.groups < least.groups || (tiled && sizes.chunks < least.chunks))
        throw KernelError("adapters: the plan does not fit the sizes that were set aside for it");
    const AdapterPlanLayout l = adapter_plan_layout(sizes);
    std::fill(out, out + l.total, 0);
    std::copy(index, index + T, out + l.token_adapter);
    const std::vector<int> slots = named(index, 0, T);
    std::vector<int> slot_of((size_t)count + 1, (int)slots.size()), fill(slots.size() + 2, 0);
    for (size_t i = 0; i < slots.size(); i++) slot_of[(size_t)slots[i]] = (int)i;
    auto slot = [&](int t) { return index[t] < 0 ? (int)slots.size() : slot_of[(size_t)index[t]]; };
    int* begin = out + l.slot_begin;
    for (int t = 0; t < T; t++) fill[(size_t)slot(t) + 1]++;
    int at = 0, g = 0, most = 0;
    for (size_t i = 0; i <= slots.size(); i++) {
        begin[i] = at;
        at += fill[i + 1];
        out[l.slot_adapter + i] = i < slots.size() ? slots[i] : -1;
        out[l.slot_group + i] = g;
        if (i < slots.size()) {
            const int n = groups_of(ranks[slots[i]]);
            for (int j = 0; j < n; j++) out[l.groups + g++] = slots[i] * ADAPTER_MAX_GROUPS + j;
            most = std::max(most, n);
        }
    }
    begin[slots.size() + 1] = T;
    out[l.slot_group + slots.size() + 1] = g;
    std::vector<int> next(begin, begin + slots.size() + 1);
    for (int t = 0; t < T; t++) {
        const int i = slot(t), place = next[(size_t)i]++;
        int* rec = out + l.places + 4 * place;
        out[l.order + place] = rec[0] = t;
        rec[1] = index[t];
        rec[2] = out[l.slot_group + i];
        rec[3] = out[l.slot_group + i + 1] - rec[2];
    }
    int chunks = 0, tile = 0;
    if (tiled && sizes.chunks > 0) {
        for (int t0 = 0; t0 < T; t0 += ADAPTER_TILE, tile++) {
            out[l.tile_chunk + tile] = chunks;
            int in = ADAPTER_CHUNK;         // groups in the last chunk
            for (int a : named(index, t0, tile_end(t0, T)))
                for (int j = 0; j < groups_of(ranks[a]); j++) {
                    if (in == ADAPTER_CHUNK) {
                        out[l.chunk_tile + chunks] = tile;
                        std::fill(out + l.chunk_groups + chunks * ADAPTER_CHUNK, out + l.chunk_groups + (chunks + 1) * ADAPTER_CHUNK, -1);
                        chunks++;
                        in = 0;
                    }
                    out[l.chunk_groups + (chunks - 1) * ADAPTER_CHUNK + in++] = a * ADAPTER_MAX_GROUPS + j;
                }
        }
        out[l.tile_chunk + tile] = chunks;
    }
    out[l.counts] = (int)slots.size();
    out[l.counts + 1] = g;
    out[l.counts + 2] = chunks;
    out[l.counts + 3] = most;
}

}  // namespace ops
}  // namespace illm
