// How the tokens of a step are divided among low-rank adapters: the plan that the host makes once per step and that the
// kernels of every projection read (adapters.cu), as one array of int32.
//
// An adapter's rank is counted in groups of 16 ("rank groups"; an adapter of rank 20 has two, the second one padded with zero
// rows).  The adapters that the step's tokens name, in ascending order, are its slots; the tokens without an adapter are a
// last slot of their own.
#pragma once

#define ADAPTER_GROUP 16          // ranks of a group: one K step of the tensor cores
#define ADAPTER_TILE 256          // tokens of a tile of the prompt product
#define ADAPTER_CHUNK 4           // groups of a chunk: one 64-wide K piece of the prompt product
#define ADAPTER_MAX_GROUPS 16     // ranks up to 256
#define ADAPTER_ROWS_MAX 128      // tokens up to which the rows form can run

struct AdapterPlanSizes {
    int T;                        // tokens
    int slots;                    // adapters named (a bound: what the arrays have room for)
    int groups;                   // rank groups of all slots (a bound)
    int chunks;                   // chunks of all tiles (a bound; 0: the plan has no tiles)
};
// Whether a step's products in bfloat16 may run as a prompt's, by tiles of tokens (the plan then has chunks): where there are more
// tokens than the rows form takes, or at least four to an adapter.
static inline bool adapter_tiled(int T, int slots) { return T > ADAPTER_ROWS_MAX || (T > 32 && 4 * slots <= T); }
// Places of the arrays in the plan; each starts on a 16-byte boundary.  The kernels read counts[1] and [2], token_adapter, places, groups
// and the tiles' arrays; the other counts and the slots' arrays say the same by slot, for whoever reads a plan on the host.
struct AdapterPlanLayout {
    int counts;                   // [4] slots, rank groups, chunks that there really are, and the most groups of a slot
    int token_adapter;            // [T] adapter of a token, -1: none
    int order;                    // [T] the tokens by slot
    int places;                   // [T * 4] per place of `order`: the token, its adapter (-1: none), where its slot begins in `groups`, how many it has
    int slot_begin;               // [slots + 2] where a slot begins in `order` (the last slot: tokens without an adapter)
    int slot_adapter;             // [slots + 1] -1 for the last
    int slot_group;               // [slots + 2] where a slot begins in `groups`
    int groups;                   // [groups] adapter * ADAPTER_MAX_GROUPS + group within the adapter
    int tile_chunk;               // [tiles + 1] where a tile of 256 tokens begins in the chunks
    int chunk_tile;               // [chunks]
    int chunk_groups;             // [chunks * 4] as `groups`, -1: none
    int total;                    // ints in all
};
static inline int adapter_pad4(int n) { return (n + 3) / 4 * 4; }
static inline AdapterPlanLayout adapter_plan_layout(const AdapterPlanSizes& s) {
    AdapterPlanLayout l;
    int off = 0;
    l.counts = off;        off += 4;
    l.token_adapter = off; off += adapter_pad4(s.T);
    l.order = off;         off += adapter_pad4(s.T);
    l.places = off;        off += s.T * 4;
    l.slot_begin = off;    off += adapter_pad4(s.slots + 2);
    l.slot_adapter = off;  off += adapter_pad4(s.slots + 1);
    l.slot_group = off;    off += adapter_pad4(s.slots + 2);
    l.groups = off;        off += adapter_pad4(s.groups);
    l.tile_chunk = off;    off += adapter_pad4((s.T + ADAPTER_TILE - 1) / ADAPTER_TILE + 1);
    l.chunk_tile = off;    off += adapter_pad4(s.chunks);
    l.chunk_groups = off;  off += s.chunks * ADAPTER_CHUNK;
    l.total = off;
    return l;
}
