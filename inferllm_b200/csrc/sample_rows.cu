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
// integer key is above the cut's, or equal and its id not above the cut's.  Nothing is sorted; a cut is found by bisection.
//
// Sums.  A vocabulary of 128k words has neighbouring partial sums nearer than float32 tells apart, and a sum whose order
// depends on timing would move a choice.  Weights are therefore made in float64 (2^(i/64) from a table times Taylor's series
// of the rest, the method of Tang, "Table-driven implementation of the exponential function", 1989; relative error below
// 2^-50) and rounded to integers in units of 2^-S with S = 62 - log2 V (at most 50): sums of integers are the same in
// every order, and are off by at most V / 2 units of 2^-S, in the mean sqrt(V) / 4 of them.
//
// One launch, a cluster of blocks per row: every block keeps its run of the row in shared memory (the row is read once), and the
// blocks exchange sums through distributed shared memory.
//   1. the largest word.  T <= 0 ends here.
//   2. a cut: a histogram over 2048 bins of the distance m - l (128 bins to an octave from 2^-8 to 2^8, whatever the
//      temperature: the bins are only a partition that keeps the order), of counts for top_k and of weights for top_p; each
//      block adds up its share of the bins for all blocks and one of them finds the bin in which the cut falls.  That bin's words
//      (some hundreds) go to the first block, which finds the cut among them, 8 bits of (value, id) at a time.  Where top_k
//      leaves at most 4096 words down to that bin, it takes all of them and finishes the row by itself.  A bin of more words
//      (many equal ones) is bisected by the whole cluster.
//   3. the kept weights' sum, then the block, the warp's run and the word in which it passes u times the whole.
#include <math.h>

#include "common.cuh"

#define SR_THREADS 512
#define SR_WARPS (SR_THREADS / 32)
#define SR_MAX_CLUSTER 8
#define SR_MAX_RESIDENT 45056       // words of a row that one block keeps
#define SR_BINS 2048
#define SR_PER 8
#define SR_LIST (SR_THREADS * SR_PER)       // words that one block takes to itself
#define SR_LIST_BITS 12

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
__device__ __forceinline__ unsigned sr_load_remote(const unsigned* local, unsigned rank) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(sr_remote(local, rank)) : "memory");
    return v;
}

// order-preserving image of a float, both zeros alike, and back
__device__ __forceinline__ unsigned sr_key(float f) {
    const unsigned u = __float_as_uint(f + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float sr_value(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
// bin of a word: 0 the nearest to the largest
__device__ __forceinline__ int sr_bin(float max_value, float l) {
    const float d = l == max_value ? 0.f : max_value - l;
    return min(max((int)(__float_as_uint(d) >> 16) - 15231, 0), SR_BINS - 1);
}

struct __align__(16) SrShared {
    double table[16];                                   // 2^(i / 16)
    u64 slot[2][SR_MAX_CLUSTER];                        // what the blocks of the cluster exchange, two in turn
    u64 found[4];                                       // what one block tells all
    u64 warp_sum[SR_WARPS];
    struct { unsigned count[256], lo[256], hi[256]; } digits[2];
    union {
        unsigned part[3][SR_BINS];                      // histogram: a sum's bits in three parts, or a count in the first
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

// A float as a double by integer instructions: the conversion instruction does 16 of them per clock and SM, a quarter of the rate
// of the float64 arithmetic behind it, and was what bound the sums.
__device__ __forceinline__ double sr_double(float f) {
    const unsigned b = __float_as_uint(f), sign = b & 0x80000000u, high = b & 0x7fffffffu;
    // zero and subnormals have no leading one: it is added with the smallest normal exponent and taken off again
    const bool small = high < 0x00800000u;
    const unsigned e = small ? 897u << 20 : 896u << 20;
    const double off = __hiloint2double((int)(small ? sign | (897u << 20) : 0u), 0);
    return __hiloint2double((int)(sign | ((high >> 3) + e)), (int)(b << 29)) - off;
}
// w of a word that can come, in units of 2^-S; 0 as well if it is below min_p (CUT).  With x = 16 (l - m) log2(e) / T = j + f, |f| <= 1/2:
// w = 2^(j / 16) exp(f ln2 / 16); the table's 16 entries lie in 32 different banks, and the series' first term left out is
// below 2^-51 of the sum.
template <bool CUT>
__device__ __forceinline__ u64 sr_weight(const SrRow& r, const double* table, float l) {
    const double x = (sr_double(l) - r.max_wide) * r.inv_temp;
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
    if (x < -1024.0) units = 0ull;                      // less than 2^-64
    return l == r.max_value ? r.one : units;
}
// whether a word can come and is still kept (no branch: the loops over the row are bound by how many of their loads and chains overlap)
__device__ __forceinline__ bool sr_kept(const SrRow& r, float l, int id) { return (l > r.low) & ((l > r.cut) | ((l == r.cut) & (id <= r.cut_id))); }

// sum over the warp by three 32-bit reductions of 22 bits each (32 of them stay below 2^27)
__device__ __forceinline__ u64 sr_warp_sum(u64 v) {
    const unsigned a = __reduce_add_sync(0xffffffffu, (unsigned)v & 0x3fffffu), b = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 22) & 0x3fffffu),
                   c = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 44));
    return (u64)a + ((u64)b << 22) + ((u64)c << 44);
}
__device__ __forceinline__ u64 sr_warp_scan(u64 v) {        // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}
// The blocks' values side by side; every thread of every block may read them in the slots that come back.  The two sets of
// slots take turns, so that a block that is behind still reads the one while the next exchange fills the other.
__device__ __forceinline__ const u64* sr_exchange(SrShared& sh, int& turn, u64 mine, int C, unsigned rank) {
    u64* s = sh.slot[turn & 1];
    turn++;
    if ((int)threadIdx.x < C) sr_store_remote(&s[rank], threadIdx.x, mine);
    sr_cluster_sync();
    return s;
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

// A list of at most SR_LIST words in ascending order of their id, dealt to the block's threads in runs: word w.at + e.
// order: key above the list's smallest key, and below it the complement of the place: larger means earlier in the row's order.
struct SrList {
    unsigned key[SR_PER];   // above the list's smallest
    unsigned least;         // that one
    int n, at;              // words of this thread, place of the first
    __device__ __forceinline__ u64 order(int e) const { return ((u64)key[e] << SR_LIST_BITS) | (unsigned)(SR_LIST - 1 - at - e); }
    __device__ __forceinline__ float value(int e) const { return sr_value(key[e] + least); }
};
// The cut of the shortest prefix, largest order first, whose measure (m[e] of word e) reaches `target`, which all of them do: kept
// are the words with order >= the result, and `last` is the smallest of them.  Digit by digit, 8 bits at a time, until a digit
// has one word.
__device__ __forceinline__ u64 sr_list_cut(SrShared& sh, const SrList& w, const u64* m, u64 target, int bits) {
    const int tid = threadIdx.x, lane = tid & 31;
    u64 prefix = 0, above = 0;
    int shift = bits;
    for (int turn = 0;; turn ^= 1) {
        unsigned *count = sh.digits[turn].count, *lo = sh.digits[turn].lo, *hi = sh.digits[turn].hi;
        for (int i = tid; i < 256; i += SR_THREADS) count[i] = lo[i] = hi[i] = 0u;
        __syncthreads();
        const int down = shift > 8 ? shift - 8 : 0, width = shift - down;
#pragma unroll
        for (int e = 0; e < SR_PER; e++)
            if (e < w.n && m[e] != 0ull && w.order(e) >> shift == prefix) {
                const int d = (int)(w.order(e) >> down) & ((1 << width) - 1);
                const unsigned low = (unsigned)m[e], carry = atomicAdd(&lo[d], low) > ~low ? 1u : 0u;
                if ((unsigned)(m[e] >> 32) + carry != 0u) atomicAdd(&hi[d], (unsigned)(m[e] >> 32) + carry);
                atomicAdd(&count[d], 1u);
            }
        __syncthreads();
        // every warp by itself: 8 digits a lane, the largest first
        u64 sum[8], mine = 0;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const int d = 255 - (lane * 8 + q);
            mine += sum[q] = ((u64)hi[d] << 32) | lo[d];
        }
        u64 before = above + sr_warp_scan(mine) - mine;
        const int owner = __ffs(__ballot_sync(0xffffffffu, before + mine >= target)) - 1;
        int digit = 0;
        bool open = true;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            if (open && before + sum[q] >= target) {
                digit = 255 - (lane * 8 + q);
                open = false;
            }
            if (open) before += sum[q];
        }
        digit = __shfl_sync(0xffffffffu, digit, owner);
        above = __shfl_sync(0xffffffffu, before, owner);
        prefix = (prefix << width) | (unsigned)digit;
        shift = down;
        if (shift == 0 || count[digit] == 1u) return prefix << shift;
    }
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

template <typename TIn>
__global__ void __launch_bounds__(SR_THREADS, 2)
sample_rows_kernel(const TIn* __restrict__ logits, long long ld, int V, int chunk, int C, int S, int part_bits, const float* __restrict__ uniforms,
                   const float* __restrict__ temps, const int* __restrict__ top_ks, const float* __restrict__ top_ps,
                   const float* __restrict__ min_ps, int* __restrict__ out) {
    extern __shared__ __align__(16) unsigned char sr_smem[];
    SrShared& sh = *reinterpret_cast<SrShared*>(sr_smem);
    float* resident = reinterpret_cast<float*>(sr_smem + sizeof(SrShared));
    unsigned* taken_mask = reinterpret_cast<unsigned*>(resident + chunk);       // a bit per word
    pdl_grid_sync();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned rank = C > 1 ? sr_rank() : 0;
    const int row = blockIdx.x / C;
    const TIn* src = logits + (long long)row * ld;
    const int first = (int)rank * chunk, n = max(0, min(V - first, chunk));     // this block's run of the row
    const int seg = ((chunk + SR_WARPS - 1) / SR_WARPS + 31) & ~31;            // a warp's run of the block's
    const int s0 = min(warp * seg, n), s1 = min(s0 + seg, n);
    if (tid < 16) sh.table[tid] = exp2((double)tid / 16.0);
    int turn = 0;
    const float temp = temps ? temps[row] : 1.0f, top_p = top_ps ? top_ps[row] : 1.0f, min_p = min_ps ? min_ps[row] : 0.f, u = uniforms[row];
    const int top_k = top_ks ? top_ks[row] : 0;
    auto value = [&](int i) { return resident[i]; };

    // 1. the row and its largest word
    float top = -INFINITY;
    {
        constexpr int W = 16 / sizeof(TIn);
        const int whole = ((uintptr_t)(src + first) & 15) == 0 ? n / W * W : 0;
#pragma unroll 4
        for (int i = tid * W; i < whole; i += SR_THREADS * W) {
            float f[W];
            if (W == 8) load8(reinterpret_cast<const bf16*>(src + first + i), f);
            else *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(src + first + i);
#pragma unroll
            for (int e = 0; e < W; e++) top = fmaxf(top, f[e]);
#pragma unroll
                for (int e = 0; e < W; e += 4) *reinterpret_cast<float4*>(resident + i + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
        }
#pragma unroll 4
        for (int i = whole + tid; i < n; i += SR_THREADS) {
            const float f = to_f32(src[first + i]);
            resident[i] = f;
            top = fmaxf(top, f);                        // (the other one of a NaN)
        }
    }
    const u64* ex = sr_exchange(sh, turn, sr_block_max(sh, sr_key(top)), C, rank);
    u64 best = 0;
    for (int c = 0; c < C; c++) best = ex[c] > best ? ex[c] : best;
    SrRow r;
    r.max_value = sr_value((unsigned)best);
    if (r.max_value == -INFINITY) {                     // nothing can come: the same in all blocks
        if (rank == 0 && tid == 0) out[row] = -1;
        return;
    }
    if (!(temp > 0.f)) {                                // the largest comes, the lowest id of equals
        unsigned least = 0;                             // its complement, for a maximum
        for (int i = tid; i < n; i += SR_THREADS)
            if (value(i) == r.max_value) { least = 0x7fffffff - (first + i); break; }
        ex = sr_exchange(sh, turn, sr_block_max(sh, least), C, rank);
        if (rank == 0 && tid == 0) {
            for (int c = 0; c < C; c++) least = max(least, (unsigned)ex[c]);
            out[row] = 0x7fffffff - (int)least;
        }
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

    auto cluster_sum = [&](u64 mine) {
        const u64* e = sr_exchange(sh, turn, sr_block_sum(sh, mine), C, rank);
        u64 t = 0;
        for (int c = 0; c < C; c++) t += e[c];
        return t;
    };
    auto tell_all = [&](int i, u64 v) {                 // by one thread
        for (int c = 0; c < C; c++) sr_store_remote(&sh.found[i], c, v);
    };
    // The first id, ascending, at which the sum of measure(i) over the ids up to it exceeds t; every thread of the cluster
    // gets it.  totals: the blocks' sums, sh.warp_sum the warps'.  The whole sum must exceed t.
    auto find = [&](u64 t, const u64* totals, auto measure) {
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
                mine = i < e ? measure(i) : 0ull;
                u64 whole;
                const u64 prior = before + sr_block_before(sh, mine, whole);
                if (prior <= t && prior + mine > t) tell_all(0, (u64)(first + i));
                before += whole;
                if (before > t) break;
            }
        }
        sr_cluster_sync();
        return (int)sh.found[0];
    };
    // The whole cluster's bisection: words with keys in [lo, hi), above = the sum over larger ones.
    auto cut_by_cluster = [&](u64 lo, u64 hi, u64 above, u64 target, auto measure) {
        while (hi - lo > 1) {
            const u64 mid = lo + (hi - lo) / 2;
            u64 mine = 0;
            for (int i = tid; i < n; i += SR_THREADS) {
                const float l = value(i);
                if (sr_kept(r, l, first + i)) {
                    const unsigned k = sr_key(l);
                    if (k >= mid && k < hi) mine += measure(l);
                }
            }
            const u64 m = cluster_sum(mine);
            if (above + m >= target) lo = mid;
            else { hi = mid; above += m; }
        }
        const float cut = sr_value((unsigned)lo);
        const u64 each = measure(cut), need = (target - above + each - 1) / each;
        auto tie = [&](int i) {
            const float l = value(i);
            return l == cut && sr_kept(r, l, first + i) ? 1ull : 0ull;
        };
        u64 mine = 0;
        for (int i = s0 + lane; i < s1; i += 32) mine += tie(i);
        const u64* totals = sr_exchange(sh, turn, sr_block_sum(sh, mine), C, rank);
        r.cut_id = find(need - 1, totals, tie);
        r.cut = cut;
    };
    // The kept words that `pick` takes, in ascending order of their id, into the first block's list; how many there are.  More
    // than the list holds: nothing is written.
    auto gather = [&](auto pick) {
        unsigned count = 0;
#pragma unroll 4
        for (int i = s0; i < s1; i += 32) {
            const float l = i + lane < s1 ? value(i + lane) : -INFINITY;
            const unsigned all = __ballot_sync(0xffffffffu, sr_kept(r, l, first + i + lane) & pick(l));
            count += __popc(all);
            if (lane == 0) taken_mask[i >> 5] = all;
        }
        const u64 block = sr_block_sum(sh, lane == 0 ? count : 0u);
        unsigned at = 0, total = 0;
#pragma unroll
        for (int q = 0; q < SR_WARPS; q++) at += q < warp ? (unsigned)sh.warp_sum[q] : 0u;
        const u64* e = sr_exchange(sh, turn, block, C, rank);
        for (int c = 0; c < C; c++) {
            if (c < (int)rank) at += (unsigned)e[c];
            total += (unsigned)e[c];
        }
        if (total > SR_LIST) return total;
        // a lane per 32 words
        for (int i0 = s0; i0 < s1 && count != 0; i0 += 1024) {
            const int i = i0 + lane * 32;
            unsigned mask = i < s1 ? taken_mask[i >> 5] : 0u;
            const unsigned mine = __popc(mask);
            unsigned run = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned v = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += v;
            }
            unsigned to = at + run - mine;
            at += __shfl_sync(0xffffffffu, run, 31);
            for (; mask; mask &= mask - 1, to++) {
                const int k = i + __ffs(mask) - 1;
                sr_store_remote(&sh.value[to], 0, __float_as_uint(value(k)));
                sr_store_remote(&sh.id[to], 0, (unsigned)(first + k));
            }
        }
        sr_cluster_sync();
        return total;
    };
    // the first block's list in its registers; `bits` how many of an order's bits differ among them
    auto take_list = [&](SrList& w, int words, int& bits) {
        const int per = (words + SR_THREADS - 1) / SR_THREADS;
        w.at = tid * per;
        w.n = max(0, min(per, words - w.at));
        unsigned most = 0, least = 0;                   // the smallest key's complement
#pragma unroll
        for (int e = 0; e < SR_PER; e++)
            if (e < w.n) {
                w.key[e] = sr_key(sh.value[w.at + e]);
                most = max(most, w.key[e]);
                least = max(least, ~w.key[e]);
            }
        most = sr_block_max(sh, most);
        w.least = ~sr_block_max(sh, least);
#pragma unroll
        for (int e = 0; e < SR_PER; e++) w.key[e] -= w.least;
        bits = 64 - __clzll(((u64)(most - w.least) << SR_LIST_BITS) | (SR_LIST - 1));
    };
    // Histogram of the kept words by bins.  Finds the bin in which the sum of measure reaches target_of(whole sum); `above` is the
    // sum over the bins before it.  false if the whole does not reach the target.
    auto bin_of = [&](auto target_of, auto measure, bool wide, int& bin, u64& above, u64& inside, u64& target) {
        for (int i = tid; i < SR_BINS; i += SR_THREADS) sh.part[0][i] = sh.part[1][i] = sh.part[2][i] = 0u;
        __syncthreads();
        const unsigned low_bits = (1u << part_bits) - 1u;
#pragma unroll 4
        for (int i = tid; i < n; i += SR_THREADS) {
            const float l = value(i);
            const u64 m = sr_kept(r, l, first + i) ? measure(l) : 0ull;
            const int b = sr_bin(r.max_value, l);
            if (!wide) {
                if (m != 0ull) atomicAdd(&sh.part[0][b], 1u);
            } else {
                const unsigned p0 = (unsigned)m & low_bits, p1 = (unsigned)(m >> part_bits) & low_bits, p2 = (unsigned)(m >> (2 * part_bits));
                if (p0) atomicAdd(&sh.part[0][b], p0);
                if (p1) atomicAdd(&sh.part[1][b], p1);
                if (p2) atomicAdd(&sh.part[2][b], p2);
            }
        }
        sr_cluster_sync();
        // this block's share of the bins, for all blocks: up to 4 neighbouring ones a thread
        const int share = SR_BINS / C, q = share < SR_THREADS ? 1 : share / SR_THREADS;
        u64 sum[SR_BINS / SR_THREADS], mine = 0;
#pragma unroll
        for (int j = 0; j < SR_BINS / SR_THREADS; j++) {
            sum[j] = 0;
            if (j < q && tid * q + j < share)
                for (int c = 0; c < C; c++) {
                    const int b = (int)rank * share + tid * q + j;
                    sum[j] += sr_load_remote(&sh.part[0][b], c);
                    if (wide) sum[j] += ((u64)sr_load_remote(&sh.part[1][b], c) << part_bits) + ((u64)sr_load_remote(&sh.part[2][b], c) << (2 * part_bits));
                }
            mine += sum[j];
        }
        const u64 block = sr_block_sum(sh, mine), *totals = sr_exchange(sh, turn, block, C, rank);
        u64 whole = 0, before = 0;
        for (int c = 0; c < C; c++) {
            if (c < (int)rank) before += totals[c];
            whole += totals[c];
        }
        target = target_of(whole);
        if (whole < target) return false;
        if (before < target && before + block >= target) {          // the block in whose share it falls
            for (int w = 0; w < warp; w++) before += sh.warp_sum[w];
            before += sr_warp_scan(mine) - mine;
#pragma unroll
            for (int j = 0; j < SR_BINS / SR_THREADS; j++) {
                if (j < q && before < target && before + sum[j] >= target) {
                    tell_all(1, (u64)((int)rank * share + tid * q + j));
                    tell_all(2, before);
                    tell_all(3, sum[j]);
                }
                before += sum[j];
            }
        }
        sr_cluster_sync();
        bin = (int)sh.found[1], above = sh.found[2], inside = sh.found[3];
        return true;
    };
    // Narrows the cut to the shortest prefix of the kept words whose measure reaches the target, given its bin.
    auto cut_in_bin = [&](int bin, u64 above, u64 target, auto measure) {
        const unsigned words = gather([&](float l) { return sr_bin(r.max_value, l) == bin; });
        if (words <= SR_LIST) {
            if (rank == 0) {
                SrList w;
                int bits;
                take_list(w, (int)words, bits);
                u64 m[SR_PER], last = ~0ull;
#pragma unroll
                for (int e = 0; e < SR_PER; e++) m[e] = e < w.n ? measure(w.value(e)) : 0ull;
                const u64 cut = sr_list_cut(sh, w, m, target - above, bits);
                // the last word of the prefix: the smallest order that is kept
#pragma unroll
                for (int e = 0; e < SR_PER; e++)
                    if (e < w.n && m[e] != 0ull && w.order(e) >= cut && w.order(e) < last) last = w.order(e);
                const unsigned high = ~sr_block_max(sh, ~(unsigned)(last >> 32)), low = ~sr_block_max(sh, (unsigned)(last >> 32) == high ? ~(unsigned)last : 0u);
#pragma unroll
                for (int e = 0; e < SR_PER; e++)
                    if (e < w.n && w.order(e) == (((u64)high << 32) | low))
                        tell_all(1, ((u64)__float_as_uint(w.value(e)) << 32) | (unsigned)sh.id[w.at + e]);
            }
            sr_cluster_sync();
            r.cut = __uint_as_float((unsigned)(sh.found[1] >> 32));
            r.cut_id = (int)(unsigned)sh.found[1];
            return;
        }
        unsigned hi = 0, lo = 0;                        // the bin's largest key, and its smallest one's complement
        for (int i = tid; i < n; i += SR_THREADS) {
            const float l = value(i);
            if (sr_kept(r, l, first + i) && sr_bin(r.max_value, l) == bin) {
                const unsigned k = sr_key(l);
                hi = max(hi, k);
                lo = max(lo, ~k);
            }
        }
        const u64* e = sr_exchange(sh, turn, sr_block_max(sh, hi), C, rank);
        for (int c = 0; c < C; c++) hi = max(hi, (unsigned)e[c]);
        e = sr_exchange(sh, turn, sr_block_max(sh, lo), C, rank);
        for (int c = 0; c < C; c++) lo = max(lo, (unsigned)e[c]);
        // (a thread's own maximum is not above the cluster's)
        cut_by_cluster((u64)~lo, (u64)hi + 1, above, target, measure);
    };
    auto one = [](float) { return 1ull; };
    auto weight_of = [&](float l) { return sr_weight<false>(r, sh.table, l); };
    int bin;
    u64 above, inside, target;

    // 2. the cuts
    if (top_k > 0 && top_k < V && bin_of([&](u64) { return (u64)top_k; }, one, false, bin, above, inside, target)) {
        if (above + inside <= SR_LIST) {
            // few words: the first block takes them all and finishes the row
            const int words = (int)gather([&](float l) { return sr_bin(r.max_value, l) <= bin; });
            if (rank != 0) return;
            SrList w;
            int bits;
            take_list(w, words, bits);
            u64 m[SR_PER], mine = 0, whole;
#pragma unroll
            for (int e = 0; e < SR_PER; e++) m[e] = e < w.n ? 1ull : 0ull;
            u64 cut = sr_list_cut(sh, w, m, target, bits);
            if (top_p < 1.0f) {
#pragma unroll
                for (int e = 0; e < SR_PER; e++) mine += m[e] = e < w.n && w.order(e) >= cut ? weight_of(w.value(e)) : 0ull;
                cut = sr_list_cut(sh, w, m, sr_top_p_target(top_p, sr_block_sum(sh, mine)), bits);
            }
            mine = 0;
#pragma unroll
            for (int e = 0; e < SR_PER; e++) mine += m[e] = e < w.n && w.order(e) >= cut ? sr_weight<true>(r, sh.table, w.value(e)) : 0ull;
            u64 before = sr_block_before(sh, mine, whole);
            const u64 t = sr_draw_target(u, whole);
            if (before <= t && before + mine > t) {
#pragma unroll
                for (int e = 0; e < SR_PER; e++) {
                    if (before <= t && before + m[e] > t) out[row] = sh.id[w.at + e];
                    before += m[e];
                }
            }
            return;
        }
        cut_in_bin(bin, above, target, one);
    }
    if (top_p < 1.0f && bin_of([&](u64 whole) { return sr_top_p_target(top_p, whole); }, weight_of, true, bin, above, inside, target))
        cut_in_bin(bin, above, target, weight_of);

    // 3. the draw
    auto weight = [&](int i) {
        const float l = value(i);
        const u64 w = sr_weight<true>(r, sh.table, l);
        return sr_kept(r, l, first + i) ? w : 0ull;
    };
    u64 mine = 0;
#pragma unroll 4
    for (int i = s0 + lane; i < s1; i += 32) mine += weight(i);
    const u64* totals = sr_exchange(sh, turn, sr_block_sum(sh, mine), C, rank);
    u64 total = 0;
    for (int c = 0; c < C; c++) total += totals[c];
    const int id = find(sr_draw_target(u, total), totals, weight);
    if (rank == 0 && tid == 0) out[row] = id;
}

template <typename TIn>
static int sr_launch(const void* logits, long long ld, int B, int V, int C, const float* u, const float* temp, const int* top_k, const float* top_p,
                     const float* min_p, int* out, cudaStream_t s) {
    const int chunk = ((V + C - 1) / C + 7) / 8 * 8;        // whole 16-byte pieces of either type
    int log_v = 0, log_chunk = 0;
    while ((1 << log_v) < V) log_v++;
    while ((1 << log_chunk) < chunk) log_chunk++;
    // a row's sum stays below 2^62; a part of the histogram, times a block's words, below 2^32
    const int part_bits = 32 - log_chunk - 1;
    int S = 62 - log_v;
    S = S > 50 ? 50 : S;
    S = S > 3 * part_bits ? 3 * part_bits : S;
    const size_t smem = sizeof(SrShared) + (size_t)chunk * sizeof(float) + (size_t)(chunk / 32 + SR_WARPS + 1) * sizeof(unsigned);
    auto kern = sample_rows_kernel<TIn>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    return illm_launch_cluster(kern, dim3((unsigned)B * C), dim3(SR_THREADS), C, smem, s, (const TIn*)logits, ld, V, chunk, C, S, part_bits, u, temp, top_k,
                               top_p, min_p, out);
}

// logits [B, V] (dtype ILLM_F32 or ILLM_BF16, rows ld elements apart), V at most 360,448; one uniform number in [0, 1) per row; temp,
// top_k, top_p and min_p [B] or nullptr (1, all, 1, 0) -> out int32 [B].
extern "C" int illm_sample_rows(const void* logits, int dtype, int B, int V, long long ld, const float* uniforms, const float* temp,
                                const int* top_k, const float* top_p, const float* min_p, int* out, void* stream) {
    if (B <= 0) return 0;
    if (V <= 0 || V > SR_MAX_CLUSTER * SR_MAX_RESIDENT || B > (1 << 24) || ld < V || !logits || !uniforms || !out) return ILLM_ERR_BAD_ARG;
    // blocks to a row: more while there are fewer than four to an SM and a block's run is worth a block, or does not fit it
    int C = 1;
    while (C < SR_MAX_CLUSTER && (((V + C - 1) / C > 2048 && (long long)B * C < 4 * illm_sm_count()) || (V + C - 1) / C > SR_MAX_RESIDENT / 2)) C *= 2;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == ILLM_F32) return sr_launch<float>(logits, ld, B, V, C, uniforms, temp, top_k, top_p, min_p, out, s);
    if (dtype == ILLM_BF16) return sr_launch<bf16>(logits, ld, B, V, C, uniforms, temp, top_k, top_p, min_p, out, s);
    return ILLM_ERR_BAD_ARG;
}
