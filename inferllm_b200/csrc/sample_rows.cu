// The next token of every row of a batch whose requests bring sampling settings of their own, from given uniform numbers.
//
// Per row, with l the logits, T the temperature and m = max l:
//   w_i  = exp((l_i - m) / T), 1 where l_i = m, 0 where l_i is -inf or NaN (such a word never comes)
//   order the words by (l descending, id ascending) and keep
//     the first top_k                                                     (top_k <= 0 or >= V: all)
//     of these the shortest prefix whose sum of w reaches top_p times theirs   (top_p >= 1: all)
//     of these the ones with w_i >= min_p                                 (min_p <= 0: all)
//   the token is the first kept id, ids ascending, at which the sum of the kept w exceeds u times their sum.
// T <= 0: the lowest id among the maxima.  A row with no word at all gives -1.
//
// All three cuts are prefixes of one order, so a cut is one pair (key, id): an element is kept if its order-preserving
// integer key is above the cut's, or equal and its id not above the cut's.  The row is not sorted: a histogram says in which bin a cut
// falls, and the bin's words are ranked (only where they are very many, a bisection takes them).
//
// Sums.  A vocabulary of 128k words has neighbouring partial sums nearer than float32 tells apart, and a sum whose order
// depends on timing would move a choice.  Weights are therefore made in float64 (2^(i/16) from a table times Taylor's series
// of the rest, the method of Tang, "Table-driven implementation of the exponential function", 1989; off by less than 2^-50 of
// the largest) and rounded to integers in units of 2^-S with S = 62 - log2 V (at most 50): sums of integers are the same in
// every order, and are off by at most V / 2 units of 2^-S, in the mean sqrt(V) / 4 of them.
//
// One launch, a cluster of blocks per row: every block keeps its run of the row in shared memory (the row is read once), and the
// blocks exchange sums through distributed shared memory.
//   1. the largest word.  T <= 0 ends here.
//   2. top_k: a histogram of counts over 2048 bins of the distance m - l (128 bins to an octave from 2^-8 to 2^8, whatever the
//      temperature: the bins are only a partition that keeps the order); the blocks tell one another the sums of 32 groups of bins,
//      then the bins of the group in which the cut falls.  Where at most 4096 words lie down to that bin (any usual top_k) the
//      first block takes them all and finishes the row by itself; otherwise it finds the cut among the bin's words.
//   3. top_p: the same histogram of float32 weights (relative to the bin's, in integers, so that their order does not matter) says
//      in which bin the cut falls, up to a rounding; one pass over the row then adds up the exact weights, all of them and those
//      before that bin, which proves the bin right or says which way to move, and notes the bin's words for the first block, which
//      finds the cut among them.
//   4. the draw: the block, the warp's run and the word in which the kept weights' sum passes u times the whole.  Behind top_p the
//      runs' sums are known from its pass.
// A bin of more than 4096 words (many equal ones) is bisected by the whole cluster.
#include <math.h>

#include "common.cuh"

#define SR_THREADS 512
#define SR_WARPS (SR_THREADS / 32)
#define SR_MAX_CLUSTER 8
#define SR_MAX_RESIDENT 45056       // words of a row that one block keeps
#define SR_BINS 2048
#define SR_GROUPS 32                // groups of bins
#define SR_GROUP (SR_BINS / SR_GROUPS)
#define SR_LIST 4096                 // words that one block takes to itself
#define SR_LIST_BITS 12
#define SR_FEW 128                  // words that are ranked by comparing each with each

typedef unsigned long long u64;

__device__ __forceinline__ unsigned sr_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void sr_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned sr_remote(const void* local, unsigned rank) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((unsigned)__cvta_generic_to_shared(local)), "r"(rank));
    return r;
}
__device__ __forceinline__ void sr_store_remote(void* local, unsigned rank, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(sr_remote(local, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void sr_store_remote(void* local, unsigned rank, unsigned v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(sr_remote(local, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void sr_store_remote(void* local, unsigned rank, float v) { sr_store_remote(local, rank, __float_as_uint(v)); }

// order-preserving image of a float, both zeros alike, and back
__device__ __forceinline__ unsigned sr_key(float f) {
    const unsigned u = __float_as_uint(f + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float sr_value(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
// distance from the largest word (0 for an infinite one), its bin (0 the nearest) and where a bin begins
__device__ __forceinline__ float sr_distance(float max_value, float l) { return l == max_value ? 0.f : max_value - l; }
__device__ __forceinline__ int sr_bin(float d) { return min(max((int)(__float_as_uint(d) >> 16) - 15231, 0), SR_BINS - 1); }
__device__ __forceinline__ float sr_edge(int bin) { return bin <= 0 ? 0.f : bin >= SR_BINS ? INFINITY : __uint_as_float((unsigned)(bin + 15231) << 16); }

struct __align__(16) SrShared {
    double table[16];                                   // 2^(i / 16)
    u64 slot[2][4][SR_MAX_CLUSTER];                     // what the blocks of the cluster exchange, two sets in turn
    u64 found;                                          // what one block tells all
    u64 warp_sum[SR_WARPS], warp_above[SR_WARPS];
    float group_sum[SR_MAX_CLUSTER][SR_GROUPS];         // every block's histogram: sums of the groups,
    float bin_sum[SR_MAX_CLUSTER][SR_GROUP];            // bins of one group
    struct { unsigned count[256], lo[256], hi[256]; } digits[2];
    u64 few_order[SR_FEW], few_weight[SR_FEW];
    unsigned n_few, few_at[SR_FEW];
    union {
        unsigned bins[SR_BINS];
        struct { float value[SR_LIST]; int id[SR_LIST]; };      // the first block's list
    };
};
static_assert(sizeof(SrShared) % 16 == 0, "the row behind it is written 16 bytes at a time");

struct SrRow {
    double inv_temp;        // 16 log2(e) / T
    double max_wide;        // max_value
    double unit;            // 2^S
    u64 one;                // 2^S
    double min_p;
    float max_value;
    float low;              // words above it can come
    float cut;              // kept: l > cut, or l == cut and id <= cut_id
    int cut_id;
};

// w of a word that can come, in units of 2^-S; 0 as well if it is below min_p (CUT).  With x = 16 (l - m) log2(e) / T = j + f, |f| <= 1/2:
// w = 2^(j / 16) exp(f ln2 / 16); the table's 16 entries lie in 32 different banks, and the series' first term left out is
// below 2^-51 of the sum.
template <bool CUT>
__device__ __forceinline__ u64 sr_weight(const SrRow& r, const double* table, float l) {
    const double x = ((double)l - r.max_wide) * r.inv_temp;
    const double shift = 6755399441055744.0;            // 1.5 * 2^52: rounds to an integer, which the low bits then hold
    const double t = x + shift;
    const int j = (int)(unsigned)__double_as_longlong(t);
    const double f = x - (t - shift);
    constexpr double c = 0.693147180559945309417 / 16.0;
    double p = c * c * c * c * c * c / 720.0;
    p = p * f + c * c * c * c * c / 120.0;
    p = p * f + c * c * c * c / 24.0;
    p = p * f + c * c * c / 6.0;
    p = p * f + c * c / 2.0;
    p = p * f + c;
    p = p * f + 1.0;
    double w = p * table[j & 15];
    w = __hiloint2double(__double2hiint(w) + ((j >> 4) << 20), __double2loint(w));
    const double two52 = 4503599627370496.0;
    u64 units = (u64)__double_as_longlong(w * r.unit + two52) & 0xFFFFFFFFFFFFFull;      // rounded to nearest
    if (CUT && w < r.min_p) units = 0ull;
    if ((unsigned)__double2hiint(x) > 0xC0900000u) units = 0ull;      // x < -1024: less than 2^-64
    return l == r.max_value ? r.one : units;
}
__device__ __forceinline__ u64 sr_measure(const SrRow& r, const double* table, float l, bool weights) { return weights ? sr_weight<false>(r, table, l) : 1ull; }
// whether a word can come and is still kept (no branch: the loops over the row are bound by how many of their loads and chains overlap)
__device__ __forceinline__ bool sr_kept(const SrRow& r, float l, int id) { return (l > r.low) & ((l > r.cut) | ((l == r.cut) & (id <= r.cut_id))); }

// sum over the warp by three 32-bit reductions of 22 bits each (32 of them stay below 2^27)
__device__ __forceinline__ u64 sr_warp_sum(u64 v) {
    const unsigned a = __reduce_add_sync(0xffffffffu, (unsigned)v & 0x3fffffu), b = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 22) & 0x3fffffu),
                   c = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 44));
    return (u64)a + ((u64)b << 22) + ((u64)c << 44);
}
template <typename T> __device__ __forceinline__ T sr_warp_scan(T v) {        // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}
// sum over the block (every thread gets it); the warps' sums stay in sh.warp_sum
__device__ __forceinline__ u64 sr_block_sum(SrShared& sh, u64 v) {
    v = sr_warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 t = 0;
#pragma unroll
    for (int w = 0; w < SR_WARPS; w++) t += sh.warp_sum[w];
    return t;
}
__device__ __forceinline__ unsigned sr_block_max(SrShared& sh, unsigned v) {
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SR_WARPS; w++) v = max(v, (unsigned)sh.warp_sum[w]);
    return v;
}
// sum over the threads before this one; `whole` gets the block's
__device__ __forceinline__ u64 sr_block_before(SrShared& sh, u64 v, u64& whole) {
    const u64 run = sr_warp_scan(v);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 31) sh.warp_sum[warp] = run;
    __syncthreads();
    u64 before = run - v;
    whole = 0;
#pragma unroll
    for (int w = 0; w < SR_WARPS; w++) {
        before += w < warp ? sh.warp_sum[w] : 0ull;
        whole += sh.warp_sum[w];
    }
    return before;
}
__device__ __forceinline__ u64 sr_top_p_target(float top_p, u64 total) {
    const u64 t = (u64)ceil((double)top_p * (double)total);
    return !(top_p > 0.f) || t == 0ull ? 1ull : t;
}
__device__ __forceinline__ u64 sr_draw_target(float u, u64 total) {
    u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;          // [0, 1); NaN counts as 0
    const u64 t = (u64)((double)u * (double)total);
    return t < total ? t : total - 1;
}

// A block's view of its row.
struct SrBlock {
    SrShared& sh;
    const float* row;       // its run of the row
    unsigned* mask;         // a bit per word of it
    int n, first, seg, s0, s1, C, tid, lane, warp;     // s0 .. s1: the warp's run of that
    unsigned rank;
    int turn;

    // The blocks' values side by side; every thread of every block may read them in the slots that come back.  The two sets of
    // slots take turns, so that a block that is behind still reads the one while the next exchange fills the other.
    template <int N> __device__ __forceinline__ const u64 (*exchange(const u64 (&mine)[N]))[SR_MAX_CLUSTER] {
        u64(*s)[SR_MAX_CLUSTER] = sh.slot[turn & 1];
        turn++;
        const int i = tid / SR_MAX_CLUSTER, c = tid % SR_MAX_CLUSTER;
#pragma unroll
        for (int j = 0; j < N; j++)
            if (i == j && c < C) sr_store_remote(&s[j][rank], c, mine[j]);
        sr_cluster_sync();
        return s;
    }
    __device__ __forceinline__ u64 cluster_sum(u64 mine) {
        const u64 m[1] = {sr_block_sum(sh, mine)};
        const u64(*e)[SR_MAX_CLUSTER] = exchange(m);
        u64 t = 0;
        for (int c = 0; c < C; c++) t += e[0][c];
        return t;
    }
    __device__ __forceinline__ unsigned cluster_max(unsigned mine) {
        const u64 m[1] = {sr_block_max(sh, mine)};
        const u64(*e)[SR_MAX_CLUSTER] = exchange(m);
        unsigned t = 0;
        for (int c = 0; c < C; c++) t = max(t, (unsigned)e[0][c]);
        return t;
    }
    __device__ __forceinline__ void tell_all(u64 v) {      // by one thread
        for (int c = 0; c < C; c++) sr_store_remote(&sh.found, c, v);
    }

    // What word i adds to a sum in ascending order of the id: its weight if it is kept, or (ties) 1 if it equals `value` and is kept.
    __device__ __forceinline__ u64 part(const SrRow& r, bool ties, float value, int i) const {
        const float l = row[i];
        const bool kept = sr_kept(r, l, first + i);
        if (ties) return (l == value) & kept ? 1ull : 0ull;
        const u64 w = sr_weight<true>(r, sh.table, l);
        return kept ? w : 0ull;
    }
    // The first id, ascending, at which the sum of part(i) over the ids up to it exceeds t; every thread of the cluster
    // gets it.  totals: the blocks' sums, sh.warp_sum the warps'.  The whole sum must exceed t.
    __device__ __forceinline__ int find(const SrRow& r, u64 t, const u64* totals, bool ties, float value) {
        u64 before = 0;
        int owner = 0;
        for (; owner < C - 1 && before + totals[owner] <= t; owner++) before += totals[owner];
        if ((int)rank == owner) {
            // the first warp whose run passes t
            u64 mine = lane < SR_WARPS ? sh.warp_sum[lane] : 0ull;
            const u64 upto = before + sr_warp_scan(mine);
            const int w = min(__ffs(__ballot_sync(0xffffffffu, upto > t)) - 1, SR_WARPS - 1);
            before = __shfl_sync(0xffffffffu, upto - mine, w);
            // the whole block over that warp's run
            const int e = min(n, (w + 1) * seg);
            for (int i0 = w * seg; i0 < e; i0 += SR_THREADS) {
                const int i = i0 + tid;
                mine = i < e ? part(r, ties, value, i) : 0ull;
                u64 whole;
                const u64 prior = before + sr_block_before(sh, mine, whole);
                if (prior <= t && prior + mine > t) tell_all((u64)(first + i));
                before += whole;
                if (before > t) break;
            }
        }
        sr_cluster_sync();
        return (int)sh.found;
    }

    // Histogram of the kept words over the bins, of counts or (WEIGHTS) of float32 weights, and the bin in which the sum reaches
    // `share` of the whole (WEIGHTS) or `share` words; `before` is the sum over the bins ahead of it, `inside` its own.  Counts
    // are exact.  false if there are fewer words.  The same in every block.
    template <bool WEIGHTS> __device__ __forceinline__ bool bin_of(const SrRow& r, float share, int part_bits, int& bin, float& before, float& inside) {
        for (int i = tid; i < SR_BINS; i += SR_THREADS) sh.bins[i] = 0u;
        __syncthreads();
        const float rate = fmaxf((float)(r.inv_temp * -0.0625), -1e30f), scale = (float)(1u << part_bits);       // log2 of a weight per distance
        const bool all = r.cut == -INFINITY;
#pragma unroll 4
        for (int i = tid; i < n; i += SR_THREADS) {
            const float l = row[i], d = sr_distance(r.max_value, l);
            const int b = sr_bin(d);
            unsigned m = 1u;
            // (2^23 as the ulp's unit: the sum's low bits are the rounded weight)
            if (WEIGHTS) m = __float_as_uint(fmaf(fast_exp2((d - sr_edge(b)) * rate), scale, 8388608.0f)) & 0x7fffffu;
            if ((l > r.low) & (all || sr_kept(r, l, first + i)) & (m != 0u)) atomicAdd(&sh.bins[b], m);
        }
        __syncthreads();
        auto mass = [&](int b) { return WEIGHTS ? (float)sh.bins[b] * fast_exp2(sr_edge(b) * rate) : (float)sh.bins[b]; };
        // groups: 16 threads each
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < SR_BINS / SR_THREADS; j++) v += mass(tid * (SR_BINS / SR_THREADS) + j);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if ((tid & 15) < C) sr_store_remote(&sh.group_sum[rank][tid >> 4], tid & 15, v);
        sr_cluster_sync();
        // every warp by itself, and alike: the group, then the bin
        v = 0.f;
        for (int c = 0; c < C; c++) v += sh.group_sum[c][lane];
        float upto = sr_warp_scan(v);
        const float whole = __shfl_sync(0xffffffffu, upto, 31), target = WEIGHTS ? share * whole : share;
        if (!WEIGHTS && whole < target) {
            // (the same in every block; the next histogram's sums go where slower warps still read these)
            sr_cluster_sync();
            return false;
        }
        auto first_lane = [&](float m) {                // where the sum reaches the target, or the last with anything in it
            const unsigned reach = __ballot_sync(0xffffffffu, (upto >= target) & (m > 0.f)), some = __ballot_sync(0xffffffffu, m > 0.f);
            return reach ? __ffs(reach) - 1 : 31 - __clz(some | 1u);
        };
        const int g = first_lane(v);
        const float ahead = __shfl_sync(0xffffffffu, upto - v, g);
        if (tid < SR_GROUP * C) sr_store_remote(&sh.bin_sum[rank][tid % SR_GROUP], tid / SR_GROUP, mass(g * SR_GROUP + tid % SR_GROUP));
        sr_cluster_sync();
        float a = 0.f, b = 0.f;
        for (int c = 0; c < C; c++) {
            a += sh.bin_sum[c][2 * lane];
            b += sh.bin_sum[c][2 * lane + 1];
        }
        upto = ahead + sr_warp_scan(a + b);
        const int p = first_lane(a + b);
        a = __shfl_sync(0xffffffffu, a, p);
        b = __shfl_sync(0xffffffffu, b, p);
        before = __shfl_sync(0xffffffffu, upto, p) - (a + b);
        const bool second = (before + a < target && b > 0.f) || !(a > 0.f);
        bin = g * SR_GROUP + 2 * p + second;
        before += second ? a : 0.f;
        inside = second ? b : a;
        return true;
    }

    // The words that a mask marks, in ascending order of their id, into the first block's list.  count: of this warp's run, at: words
    // of all runs before it.
    __device__ __forceinline__ void push(unsigned count, unsigned at) {
        // a lane per 32 words
        for (int i0 = s0; i0 < s1 && count != 0; i0 += 1024) {
            const int i = i0 + lane * 32;
            unsigned m = i < s1 ? mask[i >> 5] : 0u;
            const unsigned mine = __popc(m), run = sr_warp_scan(mine);
            unsigned to = at + run - mine;
            at += __shfl_sync(0xffffffffu, run, 31);
            for (; m; m &= m - 1, to++) {
                const int k = i + __ffs(m) - 1;
                sr_store_remote(&sh.value[to], 0, row[k]);
                sr_store_remote(&sh.id[to], 0, (unsigned)(first + k));
            }
        }
        sr_cluster_sync();
    }
    // The kept words at distances of [from, to) into the first block's list; how many there are.  More than the list holds: nothing
    // is written.
    __device__ __forceinline__ unsigned gather(const SrRow& r, float from, float to) {
        unsigned count = 0;
#pragma unroll 4
        for (int i = s0; i < s1; i += 32) {
            const float l = i + lane < s1 ? row[i + lane] : -INFINITY, d = sr_distance(r.max_value, l);
            const unsigned all = __ballot_sync(0xffffffffu, sr_kept(r, l, first + i + lane) & (d >= from) & ((d < to) | (to == INFINITY)));
            count += __popc(all);
            if (lane == 0) mask[i >> 5] = all;
        }
        const u64 m[1] = {sr_block_sum(sh, lane == 0 ? count : 0u)};
        unsigned at = 0, total = 0;
#pragma unroll
        for (int q = 0; q < SR_WARPS; q++) at += q < warp ? (unsigned)sh.warp_sum[q] : 0u;
        const u64(*e)[SR_MAX_CLUSTER] = exchange(m);
        for (int c = 0; c < C; c++) {
            if (c < (int)rank) at += (unsigned)e[0][c];
            total += (unsigned)e[0][c];
        }
        if (total <= SR_LIST) push(count, at);
        return total;
    }

    // The whole cluster's bisection among the kept words at distances of [from, to), for bins that no list holds: the cut of the
    // shortest prefix whose count, or weight, reaches `target`, `above` being that of the words before these.
    __device__ __forceinline__ void cut_by_cluster(SrRow& r, float from, float to, u64 above, u64 target, bool weights) {
        unsigned most = 0, least = 0;                   // the largest key, and the smallest one's complement
        for (int i = tid; i < n; i += SR_THREADS) {
            const float l = row[i], d = sr_distance(r.max_value, l);
            if (sr_kept(r, l, first + i) & (d >= from) & ((d < to) | (to == INFINITY))) {
                const unsigned k = sr_key(l);
                most = max(most, k);
                least = max(least, ~k);
            }
        }
        u64 hi = (u64)cluster_max(most) + 1, lo = (u64)(unsigned)~cluster_max(least);
        while (hi - lo > 1) {
            const u64 mid = lo + (hi - lo) / 2;
            u64 mine = 0;
            for (int i = tid; i < n; i += SR_THREADS) {
                const float l = row[i];
                const unsigned k = sr_key(l);
                if (sr_kept(r, l, first + i) & (k >= mid) & (k < hi)) mine += sr_measure(r, sh.table, l, weights);
            }
            const u64 m = cluster_sum(mine);
            if (above + m >= target) lo = mid;
            else { hi = mid; above += m; }
        }
        // of the words with this very value as many as are needed, in ascending order of their id
        const float cut = sr_value((unsigned)lo);
        const u64 each = sr_measure(r, sh.table, cut, weights), need = (target - above + each - 1) / each;
        u64 mine = 0;
        for (int i = s0 + lane; i < s1; i += 32) mine += part(r, true, cut, i);
        const u64 m[1] = {sr_block_sum(sh, mine)};
        const u64(*e)[SR_MAX_CLUSTER] = exchange(m);
        const int id = find(r, need - 1, e[0], true, cut);
        r.cut = cut;
        r.cut_id = id;
    }
};

// The two out of line, by value: what a function takes by its address stays in memory for the loops over the row as well.
__device__ __noinline__ int sr_find(SrBlock k, SrRow r, u64 t, const u64* totals) { return k.find(r, t, totals, false, 0.f); }
struct SrCut {
    float cut;
    int id, turn;
};
__device__ __noinline__ SrCut sr_cut_by_cluster(SrBlock k, SrRow r, float from, float to, u64 above, u64 target, bool weights) {
    k.cut_by_cluster(r, from, to, above, target, weights);
    return SrCut{r.cut, r.cut_id, k.turn};
}

// The first block's list: `words` of them in sh.value and sh.id, in ascending order of the id.  A word's order is its key above the
// list's smallest, and below that the complement of its place: larger means earlier in the row's order.
// (This part runs once per row, on one block: short code counts, since it comes from memory, not from the instruction cache.)
struct SrList {
    unsigned least;         // the smallest key
    int bits;               // of an order
};
__device__ __forceinline__ u64 sr_order(const SrShared& sh, const SrList& w, int i) {
    return ((u64)(sr_key(sh.value[i]) - w.least) << SR_LIST_BITS) | (unsigned)(SR_LIST - 1 - i);
}
__device__ __noinline__ SrList sr_list(SrShared& sh, int words) {
    unsigned most = 0, low = 0;                         // the largest key, and the smallest one's complement
#pragma unroll 1
    for (int i = threadIdx.x; i < words; i += SR_THREADS) {
        const unsigned k = sr_key(sh.value[i]);
        most = max(most, k);
        low = max(low, ~k);
    }
    most = sr_block_max(sh, most);
    const unsigned least = ~sr_block_max(sh, low);
    return SrList{least, 64 - __clzll(((u64)(most - least) << SR_LIST_BITS) | (SR_LIST - 1))};
}
// The order of the last word of the shortest prefix, largest order first, whose count, or weight, reaches `target`, among the words
// with an order of at least `from` at distances of at least `edge`; they are at most `few` and reach it.  By digits of 8 bits,
// until one holds at most 32 words, which every warp ranks by itself: a top_k's words in question are the last bin's, mostly so
// few that no digit is taken (1 to 2 us less than over the whole list, for rows with a top_k of 1000 in clusters).
__device__ __noinline__ u64 sr_list_cut(SrShared& sh, SrRow r, SrList w, int words, u64 from, float edge, int few, bool weights, u64 target) {
    const int tid = threadIdx.x, lane = tid & 31;
    u64 prefix = 0, above = 0;
    int shift = w.bits;
    // whether word i is still in question, and its order
    auto open = [&](int i, u64& o) {
        o = sr_order(sh, w, i);
        return o >= from && o >> shift == prefix && sr_distance(r.max_value, sh.value[i]) >= edge;
    };
    if (tid == 0) sh.n_few = 0;
#pragma unroll 1
    for (int turn = 0; few > 32; turn ^= 1) {
        unsigned *count = sh.digits[turn].count, *lo = sh.digits[turn].lo, *hi = sh.digits[turn].hi;
        if (tid < 256) count[tid] = lo[tid] = hi[tid] = 0u;
        __syncthreads();
        const int down = shift > 8 ? shift - 8 : 0, width = shift - down;
#pragma unroll 1
        for (int i = tid; i < words; i += SR_THREADS) {
            u64 o;
            if (!open(i, o)) continue;
            const u64 m = sr_measure(r, sh.table, sh.value[i], weights);
            const int d = (int)(o >> down) & ((1 << width) - 1);
            const unsigned low = (unsigned)m, carry = atomicAdd(&lo[d], low) > ~low ? 1u : 0u;
            if ((unsigned)(m >> 32) + carry != 0u) atomicAdd(&hi[d], (unsigned)(m >> 32) + carry);
            atomicAdd(&count[d], 1u);
        }
        __syncthreads();
        // every warp by itself: 8 digits a lane, the largest first
        u64 mine = 0;
#pragma unroll 1
        for (int q = 0; q < 8; q++) mine += ((u64)hi[255 - (lane * 8 + q)] << 32) + lo[255 - (lane * 8 + q)];
        u64 before = above + sr_warp_scan(mine) - mine;
        const int owner = __ffs(__ballot_sync(0xffffffffu, before + mine >= target)) - 1;
        int digit = 255 - lane * 8;
#pragma unroll 1
        for (int q = 0; q < 7; q++, digit--) {
            const u64 s = ((u64)hi[digit] << 32) + lo[digit];
            if (before + s >= target) break;
            before += s;
        }
        digit = __shfl_sync(0xffffffffu, digit, owner);
        above = __shfl_sync(0xffffffffu, before, owner);
        prefix = (prefix << width) | (unsigned)digit;
        shift = down;
        few = (int)count[digit];
    }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < words; i += SR_THREADS) {
        u64 o;
        if (!open(i, o)) continue;
        const unsigned to = atomicAdd(&sh.n_few, 1u);
        sh.few_order[to] = o;
        sh.few_weight[to] = sr_measure(r, sh.table, sh.value[i], weights);
    }
    __syncthreads();
    few = (int)sh.n_few;
    const u64 o = lane < few ? sh.few_order[lane] : 0ull, m = lane < few ? sh.few_weight[lane] : 0ull;
    u64 sum = above;
#pragma unroll 1
    for (int q = 0; q < few; q++) sum += sh.few_order[q] > o ? sh.few_weight[q] : 0ull;
    const int last = __ffs(__ballot_sync(0xffffffffu, lane < few && sum < target && sum + m >= target)) - 1;
    const u64 result = __shfl_sync(0xffffffffu, o, last);
    __syncthreads();                                    // (the next call begins with the counter)
    return result;
}

// The row that has this turn where rows of more work come first: those with a top_p over all words, with a top_k beyond what is
// ranked at once, any others, the ones without a random choice.  At most SR_THREADS rows.
__device__ __noinline__ int sr_row_of_turn(SrShared& sh, int B, int V, int turn, const float* temps, const int* top_ks, const float* top_ps) {
    const int row = threadIdx.x, from = min(row, B - 1), top_k = top_ks ? top_ks[from] : 0;
    const float temp = temps ? temps[from] : 1.f, top_p = top_ps ? top_ps[from] : 1.f;
    const int work = !(temp > 0.f) ? 0 : (top_k > 0) & (top_k < V) ? (top_k > SR_FEW ? 2 : 1) : top_p < 1.0f ? 3 : 1;
    // rows of every kind, 16 bits each
    u64 whole;
    const u64 before = sr_block_before(sh, row < B ? 1ull << (16 * work) : 0ull, whole);
    int at = (int)(before >> (16 * work)) & 0xffff;
    for (int w = work + 1; w < 4; w++) at += (int)(whole >> (16 * w)) & 0xffff;
    if (row < B && at == turn) sh.found = (u64)row;
    __syncthreads();
    return (int)sh.found;
}

template <typename TIn>
__global__ void __launch_bounds__(SR_THREADS, 2)
sample_rows_kernel(const TIn* __restrict__ logits, long long ld, int V, int by_work, int chunk, int C, int S, int part_bits, const float* __restrict__ uniforms,
                   const float* __restrict__ temps, const int* __restrict__ top_ks, const float* __restrict__ top_ps,
                   const float* __restrict__ min_ps, int* __restrict__ out) {
    extern __shared__ __align__(16) unsigned char sr_smem[];
    SrShared& sh = *reinterpret_cast<SrShared*>(sr_smem);
    float* resident = reinterpret_cast<float*>(sr_smem + sizeof(SrShared));
    // a block's shared memory may be written by the others of its cluster once it runs: they wait for this before the first exchange
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    pdl_grid_sync();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned rank = C > 1 ? sr_rank() : 0;
    const int turn = blockIdx.x / C, at_row = by_work ? sr_row_of_turn(sh, by_work, V, turn, temps, top_ks, top_ps) : turn;
    const TIn* src = logits + (long long)at_row * ld;
    const int first = (int)rank * chunk, n = max(0, min(V - first, chunk)), seg = ((chunk + SR_WARPS - 1) / SR_WARPS + 31) & ~31;
    const int s0 = min(warp * seg, n), s1 = min(s0 + seg, n);
    SrBlock k{sh, resident, reinterpret_cast<unsigned*>(resident + chunk), n, first, seg, s0, s1, C, tid, lane, warp, rank, 0};
    if (tid < 16) sh.table[tid] = exp2((double)tid / 16.0);
    const float temp = temps ? temps[at_row] : 1.0f, top_p = top_ps ? top_ps[at_row] : 1.0f, min_p = min_ps ? min_ps[at_row] : 0.f, u = uniforms[at_row];
    const int top_k = top_ks ? top_ks[at_row] : 0;

    // 1. the row and its largest word
    float top = -INFINITY;
    {
        constexpr int W = 16 / sizeof(TIn);
        const int whole = ((uintptr_t)(src + first) & 15) == 0 ? n / W * W : 0;
        constexpr int LOADS = 32 / W;                   // a thread's loads in flight, also where it has fewer left
#pragma unroll 1
        for (int i0 = tid * W; i0 < whole; i0 += SR_THREADS * W * LOADS) {
            uint4 raw[LOADS];
#pragma unroll
            for (int q = 0; q < LOADS; q++)
                if (i0 + q * SR_THREADS * W < whole) raw[q] = *reinterpret_cast<const uint4*>(src + first + i0 + q * SR_THREADS * W);
#pragma unroll
            for (int q = 0; q < LOADS; q++) {
                const int i = i0 + q * SR_THREADS * W;
                if (i >= whole) break;
                float f[W];
                if (W == 8) load8(reinterpret_cast<const bf16*>(&raw[q]), f);
                else *reinterpret_cast<uint4*>(f) = raw[q];
#pragma unroll
                for (int e = 0; e < W; e++) top = fmaxf(top, f[e]);
#pragma unroll
                for (int e = 0; e < W; e += 4) *reinterpret_cast<float4*>(resident + i + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
            }
        }
#pragma unroll 4
        for (int i = whole + tid; i < n; i += SR_THREADS) {
            const float f = to_f32(src[first + i]);
            resident[i] = f;
            top = fmaxf(top, f);                        // (the other one of a NaN)
        }
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    SrRow r;
    r.max_value = sr_value(k.cluster_max(sr_key(top)));
    if (r.max_value == -INFINITY) {                     // nothing can come: the same in all blocks
        if (rank == 0 && tid == 0) out[at_row] = -1;
        return;
    }
    if (!(temp > 0.f)) {                                // the largest comes, the lowest id of equals
        unsigned least = 0;                             // its complement, for a maximum
        for (int i = tid; i < n; i += SR_THREADS)
            if (resident[i] == r.max_value) { least = 0x7fffffff - (first + i); break; }
        least = k.cluster_max(least);
        if (rank == 0 && tid == 0) out[at_row] = 0x7fffffff - (int)least;
        return;
    }
    r.inv_temp = 16.0 * 1.44269504088896340736 / (double)temp;
    r.max_wide = (double)r.max_value;
    r.one = 1ull << S;
    r.unit = (double)r.one;
    r.min_p = min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0;
    r.low = r.max_value == INFINITY ? 3.402823466e38f : -INFINITY;
    r.cut = -INFINITY;
    r.cut_id = -1;
    auto cut_by_cluster = [&](float from, float to, u64 above, u64 target, bool weights) {
        const SrCut c = sr_cut_by_cluster(k, r, from, to, above, target, weights);
        r.cut = c.cut;
        r.cut_id = c.id;
        k.turn = c.turn;
    };
    // The cut among the first block's list, by that block.
    auto cut_in_list = [&](int words, bool weights, u64 target) {
        if (rank == 0) {
            const SrList w = sr_list(sh, words);
            const int i = SR_LIST - 1 - (int)(sr_list_cut(sh, r, w, words, 0ull, 0.f, words, weights, target) & (SR_LIST - 1));
            if (tid < C) sr_store_remote(&sh.found, tid, ((u64)__float_as_uint(sh.value[i]) << 32) | (unsigned)sh.id[i]);
        }
        sr_cluster_sync();
        r.cut = __uint_as_float((unsigned)(sh.found >> 32));
        r.cut_id = (int)(unsigned)sh.found;
    };
    int bin;
    float before, inside;
    u64 mine = 0;               // of this thread, of the kept words of its warp's run
    bool summed = false;

    // 2. top_k
    if (top_k > 0 && top_k < V && k.bin_of<false>(r, (float)top_k, part_bits, bin, before, inside)) {
        const float to = sr_edge(bin + 1);
        if (before + inside <= (float)SR_LIST) {
            // few words: the first block takes them all and finishes the row
            const int words = (int)k.gather(r, 0.f, to);
            if (rank != 0) return;
            const SrList w = sr_list(sh, words);
            if (words <= SR_FEW) {
                // few enough to compare each with each, 4 threads to a word
                if (tid < words) sh.few_order[tid] = sr_order(sh, w, tid);
                __syncthreads();
                const u64 o = tid / 4 < words ? sh.few_order[tid / 4] : 0ull;
                unsigned ahead = 0;
#pragma unroll 1
                for (int j = tid & 3; j < words; j += 4) ahead += sh.few_order[j] > o;
                ahead += __shfl_xor_sync(0xffffffffu, ahead, 1);
                ahead += __shfl_xor_sync(0xffffffffu, ahead, 2);
                if ((tid & 3) == 0 && tid / 4 < words) sh.few_at[ahead] = tid / 4;
                __syncthreads();
                // the words in the row's order, one to a thread, ...
                const int kept = min(top_k, words), at = tid < words ? (int)sh.few_at[tid] : -1;
                const float l = at >= 0 ? sh.value[at] : r.max_value;
                u64 m = tid < kept ? sr_weight<false>(r, sh.table, l) : 0ull, whole = 0, ahead_of = 0;
                if (top_p < 1.0f) ahead_of = sr_block_before(sh, m, whole);
                // ... their weights back into ascending order of the id
                if (at >= 0) sh.few_weight[at] = tid < kept && (top_p >= 1.0f || ahead_of < sr_top_p_target(top_p, whole)) ? sr_weight<true>(r, sh.table, l) : 0ull;
                __syncthreads();
                m = tid < words ? sh.few_weight[tid] : 0ull;
                ahead_of = sr_block_before(sh, m, whole);
                const u64 t = sr_draw_target(u, whole);
                if (ahead_of <= t && ahead_of + m > t) out[at_row] = sh.id[tid];
                return;
            }
            // (only the bin's words are in question: mostly few)
            u64 last = sr_list_cut(sh, r, w, words, 0ull, sr_edge(bin), (int)inside, false, (u64)top_k - (u64)before);
            auto sum = [&] {
                u64 mine = 0;
#pragma unroll 1
                for (int i = tid; i < words; i += SR_THREADS)
                    if (sr_order(sh, w, i) >= last) mine += sr_weight<true>(r, sh.table, sh.value[i]);
                return sr_block_sum(sh, mine);
            };
            const double min_p_given = r.min_p;
            if (top_p < 1.0f) {
                r.min_p = 0.0;                          // (it does not count for top_p's share)
                last = sr_list_cut(sh, r, w, words, last, 0.f, words, true, sr_top_p_target(top_p, sum()));
                r.min_p = min_p_given;
            }
            const u64 t = sr_draw_target(u, sum());
            u64 ahead = 0;
#pragma unroll 1
            for (int i0 = 0; i0 < words; i0 += SR_THREADS) {
                const int i = i0 + tid;
                const u64 m = i < words && sr_order(sh, w, i) >= last ? sr_weight<true>(r, sh.table, sh.value[i]) : 0ull;
                u64 whole;
                const u64 prior = ahead + sr_block_before(sh, m, whole);
                if (prior <= t && prior + m > t) out[at_row] = sh.id[i];
                ahead += whole;
            }
            return;
        }
        const float from = sr_edge(bin);
        const unsigned words = k.gather(r, from, to);
        if (words <= SR_LIST) cut_in_list((int)words, false, (u64)top_k - (u64)before);
        else cut_by_cluster(from, to, (u64)before, (u64)top_k, false);
    }

    // 3. top_p
    if (top_p < 1.0f) {
        k.bin_of<true>(r, fmaxf(top_p, 0.f), part_bits, bin, before, inside);
        u64 target;
        float from, to;
        const u64(*e)[SR_MAX_CLUSTER];
        u64 above = 0, within = 0;
        unsigned count, at, words;
        for (;;) {
            from = sr_edge(bin), to = sr_edge(bin + 1);
            u64 sum = 0, ahead = 0, own = 0;
            count = 0;
#pragma unroll 2
            for (int i = s0; i < s1; i += 32) {
                const float l = i + lane < s1 ? resident[i + lane] : -INFINITY, d = sr_distance(r.max_value, l);
                const bool kept = sr_kept(r, l, first + i + lane), here = kept & (d >= from) & ((d < to) | (to == INFINITY));
                const u64 w = sr_weight<false>(r, sh.table, l), m = kept ? w : 0ull;
                sum += m;
                ahead += d < from ? m : 0ull;
                own += here ? m : 0ull;
                const unsigned all = __ballot_sync(0xffffffffu, here);
                count += __popc(all);
                if (lane == 0) k.mask[i >> 5] = all;
            }
            u64 sums[4];
            sums[0] = sr_block_sum(sh, sum);
            sums[2] = sr_block_sum(sh, own);
            sums[3] = sr_block_sum(sh, lane == 0 ? count : 0u);
            at = 0;
#pragma unroll
            for (int q = 0; q < SR_WARPS; q++) at += q < warp ? (unsigned)sh.warp_sum[q] : 0u;
            sums[1] = sr_block_sum(sh, ahead);
            if (tid < SR_WARPS) sh.warp_above[tid] = sh.warp_sum[tid];
            e = k.exchange(sums);
            u64 total = 0;
            above = within = 0;
            words = 0;
            for (int c = 0; c < C; c++) {
                total += e[0][c];
                above += e[1][c];
                within += e[2][c];
                if (c < (int)rank) at += (unsigned)e[3][c];
                words += (unsigned)e[3][c];
            }
            target = sr_top_p_target(top_p, total);
            if (above >= target) bin--;                 // (the histogram's rounding, at a bin's border)
            else if (above + within < target) bin++;
            else break;
        }
        if (words > SR_LIST) {
            cut_by_cluster(from, to, above, target, true);
        } else {
            k.push(count, at);
            cut_in_list((int)words, true, target - above);
            if (!(min_p > 0.f)) {
                // the runs' sums: what is ahead of the bin, and the bin's words that are kept
                summed = true;
                mine = lane == 0 ? sh.warp_above[warp] : 0ull;
                for (int i0 = s0; i0 < s1 && count != 0; i0 += 1024) {
                    const int i = i0 + lane * 32;
#pragma unroll 1
                    for (unsigned m = i < s1 ? k.mask[i >> 5] : 0u; m; m &= m - 1) mine += k.part(r, false, 0.f, i + __ffs(m) - 1);
                }
            }
        }
    }

    // 4. the draw.  Words so far that min_p leaves them out are passed over without their weight (a margin of 2^-16 for the rounding).
    if (!summed) {
        float far = min_p > 0.f ? (float)(log(1.0 / r.min_p) * (double)temp) * 1.0000153f + 1e-30f : INFINITY;
        if (!(far < INFINITY)) {                        // (or an infinite temperature)
#pragma unroll 4
            for (int i = s0 + lane; i < s1; i += 32) mine += k.part(r, false, 0.f, i);
        } else {
#pragma unroll 1
            for (int i = s0; i < s1; i += 32) {
                const float l = i + lane < s1 ? resident[i + lane] : -INFINITY;
                if (sr_kept(r, l, first + i + lane) & (sr_distance(r.max_value, l) <= far)) mine += sr_weight<true>(r, sh.table, l);
            }
        }
    }
    const u64 block[1] = {sr_block_sum(sh, mine)};
    const u64(*e)[SR_MAX_CLUSTER] = k.exchange(block);
    u64 total = 0;
    for (int c = 0; c < C; c++) total += e[0][c];
    const int id = sr_find(k, r, sr_draw_target(u, total), e[0]);
    if (rank == 0 && tid == 0) out[at_row] = id;
}

template <typename TIn>
static int sr_launch(const void* logits, long long ld, int B, int V, int C, const float* u, const float* temp, const int* top_k, const float* top_p,
                     const float* min_p, int* out, cudaStream_t s) {
    const int chunk = ((V + C - 1) / C + 7) / 8 * 8;        // whole 16-byte pieces of either type
    int log_v = 0, log_chunk = 0;
    while ((1 << log_v) < V) log_v++;
    while ((1 << log_chunk) < chunk) log_chunk++;
    // a row's sum stays below 2^62; a bin's float32 weights in units of 2^-part_bits, a block's words at most, below 2^32
    const int part_bits = log_chunk > 9 ? 31 - log_chunk : 22, S = log_v > 12 ? 62 - log_v : 50;
    const size_t smem = sizeof(SrShared) + (size_t)chunk * sizeof(float) + (size_t)(chunk / 32 + SR_WARPS + 1) * sizeof(unsigned);
    auto kern = sample_rows_kernel<TIn>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    // More blocks than run at once, in few rounds: the rows of much work first.  64 mixed rows of 128,256 words 59 us instead of 67, 256
    // of 32,000 51 instead of 63; rows that are all alike lose 2 to 4 us in finding their turns.
    const int by_work = (long long)B * C > 2 * illm_sm_count() && B <= SR_THREADS && (top_k || top_p) ? B : 0;
    return illm_launch_cluster(kern, dim3((unsigned)B * C), dim3(SR_THREADS), C, smem, s, (const TIn*)logits, ld, V, by_work, chunk, C, S, part_bits, u, temp, top_k,
                               top_p, min_p, out);
}

// logits [B, V] (dtype ILLM_F32 or ILLM_BF16, rows ld elements apart), V at most 360,448; one uniform number in [0, 1) per row; temp,
// top_k, top_p and min_p [B] or nullptr (1, all, 1, 0) -> out int32 [B].
extern "C" int illm_sample_rows(const void* logits, int dtype, int B, int V, long long ld, const float* uniforms, const float* temp,
                                const int* top_k, const float* top_p, const float* min_p, int* out, void* stream) {
    if (B <= 0) return 0;
    if (V <= 0 || V > SR_MAX_CLUSTER * SR_MAX_RESIDENT || B > (1 << 24) || ld < V || !logits || !uniforms || !out) return ILLM_ERR_BAD_ARG;
    // blocks to a row: more while there are fewer than two to an SM (which is what its registers hold) and a block's run is worth a
    // block, or is more than two of them on an SM can keep.  Mixed settings, a replayed graph behind a flush of L2: 256 rows of 32,000
    // words (bfloat16) on 1, 2, 4, 8 blocks each 69, 52, 65, 106 us; one row 25, 21, 16, 16; 64 rows of 128,256 words on 4 and 8 73 and
    // 55; 16 rows of as many, temperature alone, 25 on both.
    int C = 1;
    while (C < SR_MAX_CLUSTER && (((V + C - 1) / C > 2048 && (long long)B * C < 2 * illm_sm_count()) || (V + C - 1) / C > SR_MAX_RESIDENT / 2)) C *= 2;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == ILLM_F32) return sr_launch<float>(logits, ld, B, V, C, uniforms, temp, top_k, top_p, min_p, out, s);
    if (dtype == ILLM_BF16) return sr_launch<bf16>(logits, ld, B, V, C, uniforms, temp, top_k, top_p, min_p, out, s);
    return ILLM_ERR_BAD_ARG;
}

// The repetition penalty of rows with settings of their own: a block per row, a thread per word of its last ones, each word once.
__global__ void __launch_bounds__(128) penalise_kernel(float* __restrict__ logits, int V, const int* __restrict__ last, int n_last, const float* __restrict__ penalty) {
    pdl_grid_sync();
    const float p = penalty[blockIdx.x];
    const int* mine = last + (size_t)blockIdx.x * n_last;
    float* row = logits + (size_t)blockIdx.x * V;
    if (p == 1.0f) return;
    for (int j = threadIdx.x; j < n_last; j += 128) {
        const int id = mine[j];
        if (id < 0 || id >= V) continue;
        bool first = true;
        for (int e = 0; e < j && first; e++) first = mine[e] != id;
        if (first) row[id] = row[id] < 0.f ? row[id] * p : row[id] / p;
    }
}
extern "C" int illm_penalise(float* logits, int B, int V, const int* last, int n_last, const float* penalty, void* stream) {
    if (B <= 0 || n_last <= 0) return 0;
    if (V <= 0 || !logits || !last || !penalty) return ILLM_ERR_BAD_ARG;
    illm_launch(penalise_kernel, dim3((unsigned)B), dim3(128), 0, (cudaStream_t)stream, logits, V, last, n_last, penalty);
    return illm_launch_status();
}
