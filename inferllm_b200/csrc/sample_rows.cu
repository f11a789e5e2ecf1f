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
// 2^-52) and rounded to integers in units of 2^-S with S = 62 - log2 V (at most 50): sums of integers are the same in
// every order, and are off by at most V / 2 units of 2^-S, in the mean sqrt(V) / 4 of them.
//
// One cluster of blocks per row: every block keeps its run of the row in shared memory (the row is read once), and the
// blocks exchange sums through distributed shared memory.  Rows too long for that are read again where they are needed.
#include <math.h>

#include "common.cuh"

#define SR_THREADS 512
#define SR_WARPS (SR_THREADS / 32)
#define SR_MAX_CLUSTER 8
#define SR_MAX_RESIDENT 51200       // words of a row that one block keeps

__device__ __forceinline__ unsigned sr_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void sr_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void sr_store_remote(void* local, unsigned rank, unsigned long long v) {
    unsigned a = (unsigned)__cvta_generic_to_shared(local), r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(r), "l"(v) : "memory");
}

// order-preserving image of a float; 0 for words that cannot come (-inf, NaN), both zeros alike
__device__ __forceinline__ unsigned sr_key(float f) {
    const unsigned u = __float_as_uint(f + 0.0f);
    const unsigned k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return f > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float sr_value(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

struct SrShared {
    double table[64];                                   // 2^(i / 64)
    unsigned long long slot[2][SR_MAX_CLUSTER];         // what the blocks of the cluster exchange, two in turn
    unsigned long long found;
    unsigned long long warp_sum[SR_WARPS];
    unsigned long long block_total;
};

struct SrRow {
    double inv_temp;        // log2(e) / T
    double max_value;
    double unit;            // 2^S
    double min_p;
    unsigned cut_key;       // kept: key > cut_key, or key == cut_key and id <= cut_id
    int cut_id;
};

// w of a present word, in units of 2^-S; 0 as well if it is below min_p (CUT)
template <bool CUT>
__device__ __forceinline__ unsigned long long sr_weight(const SrRow& r, const double* table, float l) {
    const double d = (double)l - r.max_value;           // NaN for two infinities: their weight is 1
    const double y = d * r.inv_temp;
    if (y < -64.0 || d == -INFINITY) return 0ull;
    double w = 1.0;
    if (y < 0.0) {
        const double shift = 6755399441055744.0;        // 1.5 * 2^52: rounds to an integer, which the low bits then hold
        const double t = y * 64.0 + shift;
        const int j = (int)(unsigned)__double_as_longlong(t);
        const double z = (y - (t - shift) * (1.0 / 64.0)) * 0.693147180559945309417;
        double p = 1.0 / 120.0;
        p = p * z + 1.0 / 24.0;
        p = p * z + 1.0 / 6.0;
        p = p * z + 0.5;
        p = p * z + 1.0;
        p = p * z + 1.0;
        w = p * table[j & 63];
        w = __hiloint2double(__double2hiint(w) + ((j >> 6) << 20), __double2loint(w));
    }
    if (CUT && w < r.min_p) return 0ull;
    const double two52 = 4503599627370496.0;
    return (unsigned long long)__double_as_longlong(w * r.unit + two52) & 0xFFFFFFFFFFFFFull;      // rounded to nearest
}
__device__ __forceinline__ bool sr_kept(const SrRow& r, unsigned key, int id) { return key > r.cut_key || (key == r.cut_key && id <= r.cut_id); }

__device__ __forceinline__ unsigned long long sr_warp_sum(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The blocks' values side by side; every thread of every block may read them in the slots that come back.  The two sets of
// slots take turns, so that a block that is behind still reads the one while the next exchange fills the other.
__device__ __forceinline__ const unsigned long long* sr_exchange(SrShared& sh, int& turn, unsigned long long mine, int C, unsigned rank) {
    unsigned long long* s = sh.slot[turn & 1];
    turn++;
    if ((int)threadIdx.x < C) sr_store_remote(&s[rank], threadIdx.x, mine);
    sr_cluster_sync();
    return s;
}
// sum over the block (every thread gets it); the warps' sums stay in sh.warp_sum
__device__ __forceinline__ unsigned long long sr_block_sum(SrShared& sh, unsigned long long v) {
    v = sr_warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long t = 0;
#pragma unroll
    for (int w = 0; w < SR_WARPS; w++) t += sh.warp_sum[w];
    return t;
}

template <typename TIn, bool RESIDENT>
__global__ void __launch_bounds__(SR_THREADS)
sample_rows_kernel(const TIn* __restrict__ logits, long long ld, int V, int chunk, int C, int S, const float* __restrict__ uniforms,
                   const float* __restrict__ temps, const int* __restrict__ top_ks, const float* __restrict__ top_ps,
                   const float* __restrict__ min_ps, int* __restrict__ out) {
    extern __shared__ float resident[];
    __shared__ SrShared sh;
    pdl_grid_sync();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned rank = C > 1 ? sr_rank() : 0;
    const int row = blockIdx.x / C;
    const TIn* src = logits + (long long)row * ld;
    const int first = (int)rank * chunk, n = max(0, min(V - first, chunk));     // this block's run of the row
    const int seg = ((chunk + SR_WARPS - 1) / SR_WARPS + 31) & ~31;            // a warp's run of the block's
    const int s0 = min(warp * seg, n), s1 = min(s0 + seg, n);
    if (tid < 64) sh.table[tid] = exp2((double)tid / 64.0);
    int turn = 0;

    // the row, its largest word and the smallest
    unsigned top = 0u, bottom = 0xffffffffu;
    int top_id = 0x7fffffff;
    for (int i = s0 + lane; i < s1; i += 32) {
        const float f = to_f32(src[first + i]);
        if (RESIDENT) resident[i] = f;
        const unsigned k = sr_key(f);
        if (k > top) { top = k; top_id = first + i; }
        if (k != 0u && k < bottom) bottom = k;
    }
    // (largest key, lowest id) as one number: the id's complement in the low half
    unsigned long long best = ((unsigned long long)top << 32) | (unsigned)(0x7fffffff - top_id);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long b2 = __shfl_xor_sync(0xffffffffu, best, o);
        best = b2 > best ? b2 : best;
    }
    bottom = __reduce_min_sync(0xffffffffu, bottom);
    if (lane == 0) sh.warp_sum[warp] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SR_WARPS; w++) best = sh.warp_sum[w] > best ? sh.warp_sum[w] : best;
    __syncthreads();
    if (lane == 0) sh.warp_sum[warp] = bottom;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SR_WARPS; w++) bottom = min(bottom, (unsigned)sh.warp_sum[w]);
    const unsigned long long* ex = sr_exchange(sh, turn, best, C, rank);
    for (int c = 0; c < C; c++) best = ex[c] > best ? ex[c] : best;
    ex = sr_exchange(sh, turn, bottom, C, rank);
    for (int c = 0; c < C; c++) bottom = min(bottom, (unsigned)ex[c]);
    const unsigned max_key = (unsigned)(best >> 32);
    const float temp = temps ? temps[row] : 1.0f;
    if (max_key == 0u || !(temp > 0.f)) {               // nothing can come, or the largest comes: the same in all blocks
        if (rank == 0 && tid == 0) out[row] = max_key == 0u ? -1 : 0x7fffffff - (int)(unsigned)best;
        return;
    }

    SrRow r;
    r.max_value = (double)sr_value(max_key);
    r.inv_temp = 1.44269504088896340736 / (double)temp;
    r.unit = (double)(1ull << S);
    const float min_p = min_ps ? min_ps[row] : 0.f;
    r.min_p = min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0;
    r.cut_key = 0u;
    r.cut_id = -1;

    auto value = [&](int i) { return RESIDENT ? resident[i] : to_f32(src[first + i]); };
    auto cluster_sum = [&](unsigned long long mine) {
        mine = sr_block_sum(sh, mine);
        const unsigned long long* e = sr_exchange(sh, turn, mine, C, rank);
        unsigned long long t = 0;
        for (int c = 0; c < C; c++) t += e[c];
        return t;
    };
    // The first id, ascending, at which the sum of measure(i) over the ids up to it exceeds t; every thread of the cluster
    // gets it.  The whole sum must exceed t.
    auto find = [&](unsigned long long mine, unsigned long long t, const unsigned long long* totals, auto measure) {
        unsigned long long before = 0;
        int owner = 0;
        for (; owner < C - 1 && before + totals[owner] <= t; owner++) before += totals[owner];
        if ((int)rank == owner) {
            for (int w = 0; w < SR_WARPS; w++) {
                const unsigned long long ws = sh.warp_sum[w];
                if (before + ws > t) {
                    if (warp == w) {
                        int at = -1;
                        for (int i0 = s0; i0 < s1 && at < 0; i0 += 32) {
                            unsigned long long run = i0 + lane < s1 ? measure(i0 + lane) : 0ull;
#pragma unroll
                            for (int o = 1; o < 32; o <<= 1) {
                                const unsigned long long v = __shfl_up_sync(0xffffffffu, run, o);
                                if (lane >= o) run += v;
                            }
                            const unsigned over = __ballot_sync(0xffffffffu, before + run > t);
                            if (over) at = i0 + __ffs(over) - 1;
                            before += __shfl_sync(0xffffffffu, run, 31);
                        }
                        if (lane < C) sr_store_remote(&sh.found, lane, (unsigned long long)(first + at));
                    }
                    break;
                }
                before += ws;
            }
        }
        sr_cluster_sync();
        return (int)sh.found;
    };
    // Narrows the cut to the shortest prefix of the kept words, in the row's order, whose sum of measure(key, i) reaches
    // `target` (which the sum over all of them does).
    auto cut_at = [&](unsigned long long target, auto measure) {
        unsigned long long lo = bottom, hi = (unsigned long long)max_key + 1, above = 0;       // sum over keys >= hi: above < target
        while (hi - lo > 1) {
            const unsigned mid = (unsigned)(lo + (hi - lo) / 2);
            unsigned long long mine = 0;
            for (int i = s0 + lane; i < s1; i += 32) {
                const float l = value(i);
                const unsigned k = sr_key(l);
                if (k >= mid && k < hi && sr_kept(r, k, first + i)) mine += measure(l);
            }
            const unsigned long long m = cluster_sum(mine);
            if (above + m >= target) lo = mid;
            else { hi = mid; above += m; }
        }
        // of the words with this very key as many as are needed, in ascending order of their id
        const unsigned key = (unsigned)lo;
        const unsigned long long each = measure(sr_value(key));
        const unsigned long long need = (target - above + each - 1) / each;
        unsigned long long mine = 0;
        auto tie = [&](int i) {
            const unsigned k = sr_key(value(i));
            return (k == key && sr_kept(r, k, first + i)) ? 1ull : 0ull;
        };
        for (int i = s0 + lane; i < s1; i += 32) mine += tie(i);
        mine = sr_block_sum(sh, mine);
        const unsigned long long* totals = sr_exchange(sh, turn, mine, C, rank);
        const int id = find(mine, need - 1, totals, tie);
        r.cut_key = key;
        r.cut_id = id;
    };

    const int top_k = top_ks ? top_ks[row] : 0;
    if (top_k > 0 && top_k < V) {
        unsigned long long mine = 0;
        for (int i = s0 + lane; i < s1; i += 32) mine += sr_key(value(i)) != 0u;
        if (cluster_sum(mine) > (unsigned long long)top_k) cut_at((unsigned long long)top_k, [&](float) { return 1ull; });
    }
    const float top_p = top_ps ? top_ps[row] : 1.0f;
    if (top_p < 1.0f) {
        unsigned long long mine = 0;
        for (int i = s0 + lane; i < s1; i += 32) {
            const float l = value(i);
            const unsigned k = sr_key(l);
            if (k != 0u && sr_kept(r, k, first + i)) mine += sr_weight<false>(r, sh.table, l);
        }
        const double total = (double)cluster_sum(mine);
        unsigned long long target = (unsigned long long)ceil((double)top_p * total);
        if (!(top_p > 0.f) || target == 0ull) target = 1ull;
        cut_at(target, [&](float l) { return sr_weight<false>(r, sh.table, l); });
    }
    auto weight = [&](int i) {
        const float l = value(i);
        const unsigned k = sr_key(l);
        return k != 0u && sr_kept(r, k, first + i) ? sr_weight<true>(r, sh.table, l) : 0ull;
    };
    unsigned long long mine = 0;
    for (int i = s0 + lane; i < s1; i += 32) mine += weight(i);
    mine = sr_block_sum(sh, mine);
    const unsigned long long* totals = sr_exchange(sh, turn, mine, C, rank);
    unsigned long long total = 0;
    for (int c = 0; c < C; c++) total += totals[c];
    float u = uniforms[row];
    u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;          // [0, 1); NaN counts as 0
    const unsigned long long t = (unsigned long long)((double)u * (double)total);
    const int id = find(mine, t < total ? t : total - 1, totals, weight);
    if (rank == 0 && tid == 0) out[row] = id;
}

template <typename TIn, bool RESIDENT>
static int sr_launch(const void* logits, long long ld, int B, int V, int C, const float* u, const float* temp, const int* top_k, const float* top_p,
                     const float* min_p, int* out, cudaStream_t s) {
    int S = 62;
    while (S > 0 && (1ll << (62 - S)) < V) S--;
    if (S > 50) S = 50;
    const int chunk = (V + C - 1) / C;
    const size_t smem = RESIDENT ? (size_t)chunk * sizeof(float) : 0;
    auto kern = sample_rows_kernel<TIn, RESIDENT>;
    if (smem > 40 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
    }
    return illm_launch_cluster(kern, dim3((unsigned)B * C), dim3(SR_THREADS), C, smem, s, (const TIn*)logits, ld, V, chunk, C, S, u, temp, top_k, top_p,
                               min_p, out);
}

// logits [B, V] (dtype ILLM_F32 or ILLM_BF16, rows ld elements apart), one uniform number in [0, 1) per row; temp, top_k, top_p and
// min_p [B] or nullptr (1, all, 1, 0) -> out int32 [B].
extern "C" int illm_sample_rows(const void* logits, int dtype, int B, int V, long long ld, const float* uniforms, const float* temp,
                                const int* top_k, const float* top_p, const float* min_p, int* out, void* stream) {
    if (B <= 0) return 0;
    if (V <= 0 || V > 0x7ffffff0 || B > (1 << 24) || ld < V || !logits || !uniforms || !out) return ILLM_ERR_BAD_ARG;
    int C = 1;
    while (C < SR_MAX_CLUSTER && (V + C - 1) / C > 4096) C *= 2;
    const bool resident = (V + C - 1) / C <= SR_MAX_RESIDENT;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == ILLM_F32)
        return resident ? sr_launch<float, true>(logits, ld, B, V, C, uniforms, temp, top_k, top_p, min_p, out, s)
                        : sr_launch<float, false>(logits, ld, B, V, C, uniforms, temp, top_k, top_p, min_p, out, s);
    if (dtype == ILLM_BF16)
        return resident ? sr_launch<bf16, true>(logits, ld, B, V, C, uniforms, temp, top_k, top_p, min_p, out, s)
                        : sr_launch<bf16, false>(logits, ld, B, V, C, uniforms, temp, top_k, top_p, min_p, out, s);
    return ILLM_ERR_BAD_ARG;
}
