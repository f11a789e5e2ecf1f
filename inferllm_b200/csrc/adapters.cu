// Low-rank adapters of many requests beside a shared projection:
//   y[t] = x[t] W^T + s_a (x[t] A_a^T) B_a^T,   a the adapter of token t's request, or none.
// x [T, K], W [N, K]; the adapters of a projection lie in one piece: A [count, R, K] and B [count, R / 16, N, 16] (the second
// factor by groups of 16 ranks, so that one K step of a tensor-core product, or 32 to 64 bytes of one output, lie together),
// R the largest rank rounded up to 16, rows beyond an adapter's own rank zero and, where they fill a group, never read.
// Which token has which adapter comes as a plan (adapters.h).
//
// Float32: the package's product, which adds up every output in one chain over K, then
//   shrink   v[t] = s_a x[t] A_a^T: a block per 4 tokens of the plan's order and rank group, a warp per two ranks, which
//            reads a row of A once for the tokens of a slot;
//   expand   y[t, n] += v[t] . B_a[n]: a thread per output column, 16 values of B in registers for neighbours with one adapter.
// A token's sums have one order whatever else is in the batch, and one without an adapter keeps the plain product's bits.
// 257 tokens of 1024 x 5632: 97 us of product (bound by its FMAs: 41 at full rate, and three rounds of tiles), 12 of adapters.
// Bfloat16: token by token below, tiles of tokens in adapters_prompt.cu (ad_tiled).
#include "adapters.cuh"
#include "kernels.h"

#define AD_TOKENS 8
#define AD_SHRINK 4
#define AD_COLS 128

// v[t, 16 g + r] for the ranks of group g of token t's adapter, float32 [T, R]; W floats of a row at a time
template <int W>
__global__ void __launch_bounds__(256)
adapter_shrink_kernel(const float* __restrict__ x, int K, const float* __restrict__ a, const float* __restrict__ scales, int R, const int4* __restrict__ places,
                      int tokens, float* __restrict__ v) {
    pdl_grid_sync();
    const int lane = threadIdx.x & 31, rank = blockIdx.y * ADAPTER_GROUP + (threadIdx.x >> 5) * 2, p0 = blockIdx.x * AD_SHRINK;
    for (int i = 0; i < AD_SHRINK;) {
        if (p0 + i >= tokens) return;
        // the neighbours with this token's adapter share its rows
        const int4 at = places[p0 + i];
        if (at.y < 0) return;                           // the rest has no adapter
        int n = 1;
        while (i + n < AD_SHRINK && p0 + i + n < tokens && places[p0 + i + n].y == at.y) n++;
        if ((int)blockIdx.y < at.w) {
            const float* a0 = a + ((long long)at.y * R + rank) * K;
            const float* xr[AD_SHRINK];
            float acc[2][AD_SHRINK];
#pragma unroll
            for (int e = 0; e < AD_SHRINK; e++) {
                xr[e] = x + (long long)places[p0 + i + min(e, n - 1)].x * K;
                acc[0][e] = acc[1][e] = 0.f;
            }
#pragma unroll 2
            for (int k = lane * W; k < K; k += 32 * W) {
                float w0[W], w1[W], f[W];
                AdColumns<W>::load(a0 + k, w0);
                AdColumns<W>::load(a0 + K + k, w1);
#pragma unroll
                for (int e = 0; e < AD_SHRINK; e++) {
                    AdColumns<W>::load(xr[e] + k, f);
#pragma unroll
                    for (int q = 0; q < W; q++) {
                        acc[0][e] = fmaf(f[q], w0[q], acc[0][e]);
                        acc[1][e] = fmaf(f[q], w1[q], acc[1][e]);
                    }
                }
            }
            const float s = scales[at.y];
#pragma unroll
            for (int e = 0; e < AD_SHRINK; e++) {
                const float s0 = warp_sum(acc[0][e]), s1 = warp_sum(acc[1][e]);
                if (lane == 0 && e < n) {
                    float* to = v + (long long)places[p0 + i + e].x * R + rank;
                    to[0] = s * s0;
                    to[1] = s * s1;
                }
            }
        }
        i += n;
    }
}

// out[t, n] += v[t] . B_a[n]
__global__ void __launch_bounds__(AD_COLS)
adapter_expand_kernel(int N, const float* __restrict__ b, const float* __restrict__ v, int R, const int4* __restrict__ places, int tokens, float* out) {
    pdl_grid_sync();
    const int col = blockIdx.x * AD_COLS + threadIdx.x, p0 = blockIdx.y * AD_TOKENS;
    if (col >= N) return;
    int4 at[AD_TOKENS];
    float acc[AD_TOKENS];
    int most = 0;
#pragma unroll
    for (int i = 0; i < AD_TOKENS; i++) {
        at[i] = p0 + i < tokens ? places[p0 + i] : make_int4(-1, -1, 0, 0);
        most = max(most, at[i].w);
        acc[i] = at[i].w > 0 ? out[(long long)at[i].x * N + col] : 0.f;
    }
    for (int g = 0; g < most; g++) {
        float w[ADAPTER_GROUP];
#pragma unroll
        for (int i = 0; i < AD_TOKENS; i++)
            if (g < at[i].w) {
                if (i == 0 || at[i].y != at[i - 1].y) {
                    const float* bw = b + (((long long)at[i].y * (R / ADAPTER_GROUP) + g) * N + col) * ADAPTER_GROUP;
                    load8(bw, w);
                    load8(bw + 8, w + 8);
                }
                const float* vt = v + (long long)at[i].x * R + g * ADAPTER_GROUP;
#pragma unroll
                for (int r = 0; r < ADAPTER_GROUP; r++) acc[i] = fmaf(vt[r], w[r], acc[i]);
            }
    }
#pragma unroll
    for (int i = 0; i < AD_TOKENS; i++)
        if (at[i].w > 0) out[(long long)at[i].x * N + col] = acc[i];
}

// ---- The rows form (bfloat16, up to 128 tokens): two launches.
//
// The first streams W once and, in the same grid, the first factors of the adapters that the tokens name: rank groups are
// nothing but more rows of the weight.  A block multiplies 128 of those rows (a tile of W, or 8 rank groups fetched by a TMA box
// of 16 rows each, so that they may come from any adapters) with all tokens over its slice of K on tcgen05, the rows on the
// 128 lanes, the tokens as the MMA's N, and leaves float32 slices, so that all SMs stream whatever N is.
// The second adds up the slices and, in the same float32 sum, v[t] . B_a[n]; v, the tokens' rank values, is added up and
// scaled by every block for the tokens that it works on.  It stays float32: the result is rounded once.
// Bound: reading the weight and the factors, and two starts and ends.  One token of 4096 x 4096 9.9 us on the GPU (the weight's 33 MB
// at the copy rate: 5.1), 8 tokens with 8 adapters of 4096 x 12288 22.6 (16.0), 64 tokens with 48 of 11008 x 4096 33.2 (19.4).
#define AD_ROWS_MAX_STAGES 8

template <int BN>
__global__ void __launch_bounds__(TC_THREADS)
adapter_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_x,
                    float* __restrict__ base, float* __restrict__ vs, int v_ld, int T, int N, int R, int base_tiles, const AdPlan plan, int k_iters_total,
                    int k_iters_per_split, int STAGES, int early, int* __restrict__ err) {
    constexpr unsigned A_BYTES = TC_BM * TC_BK * 2, B_BYTES = BN * TC_BK * 2, BOX_BYTES = ADAPTER_GROUP * TC_BK * 2;
    constexpr unsigned TMEM_COLS = BN < 32 ? 32 : BN;
    constexpr unsigned IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(BN >> 3) << 17) | ((unsigned)(TC_BM >> 4) << 24);
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * AD_ROWS_MAX_STAGES + 1];
    __shared__ unsigned tmem_holder;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool shrink = (int)blockIdx.x >= base_tiles;
    const int g0 = shrink ? ((int)blockIdx.x - base_tiles) * (TC_BM / ADAPTER_GROUP) : 0;
    int boxes = 0;
    if (shrink) {
        boxes = min(TC_BM / ADAPTER_GROUP, plan.counts[1] - g0);
        if (boxes <= 0) return;                         // the grid is sized for more rank groups than there are
    }
    const int ra0 = blockIdx.x * TC_BM, rows = shrink ? boxes * ADAPTER_GROUP : min(TC_BM, N - ra0);

    const unsigned a_base = (tc_smem_u32(smem_raw) + 1023u) & ~1023u, b_base = a_base + STAGES * A_BYTES;
    const unsigned full0 = tc_smem_u32(&bars[0]), empty0 = tc_smem_u32(&bars[AD_ROWS_MAX_STAGES]);
    const unsigned done_bar = tc_smem_u32(&bars[2 * AD_ROWS_MAX_STAGES]);
    const int k_begin = blockIdx.z * k_iters_per_split, n_k = min(k_iters_total - k_begin, k_iters_per_split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        mbar_init(done_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(&tmem_holder)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_holder;

    // (the two warps stay together around what one lane issues: what every lane agrees on then lies in uniform registers)
    if (warp == 0) {
        const bool elected = elect_one();
        // the join reads second factors before its wait: not before this kernel's own wait, unless no kernel before made them
        if (early) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        int group_row[TC_BM / ADAPTER_GROUP];
#pragma unroll
        for (int j = 0; j < TC_BM / ADAPTER_GROUP; j++) {
            const int g = j < boxes ? plan.groups[g0 + j] : 0;
            group_row[j] = (g / ADAPTER_MAX_GROUPS) * R + (g % ADAPTER_MAX_GROUPS) * ADAPTER_GROUP;
        }
        auto arm_and_load_weights = [&](int i, int s) {
            mbar_expect_tx(full0 + 8 * s, (shrink ? boxes * BOX_BYTES : A_BYTES) + B_BYTES);
            const int kx = (k_begin + i) * TC_BK;
            if (!shrink) {
                tma_load_2d(a_base + s * A_BYTES, &map_w, kx, ra0, full0 + 8 * s);
            } else {
#pragma unroll
                for (int j = 0; j < TC_BM / ADAPTER_GROUP; j++)
                    if (j < boxes) tma_load_2d(a_base + s * A_BYTES + j * BOX_BYTES, &map_a, kx, group_row[j], full0 + 8 * s);
            }
        };
        // where no kernel before this one makes weights, the first ring of them comes before the wait for the tokens' rows
        const int n_pre = n_k < STAGES ? n_k : STAGES;
        if (!early) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        }
        if (elected)
            for (int i = 0; i < n_pre; i++) arm_and_load_weights(i, i);
        if (early) asm volatile("griddepcontrol.wait;" ::: "memory");
        if (elected)
            for (int i = 0; i < n_pre; i++) tma_load_2d(b_base + i * B_BYTES, &map_x, (k_begin + i) * TC_BK, 0, full0 + 8 * i);
        bool alive = true;
        int s = 0, phase = 0;
        for (int i = n_pre; i < n_k; i++) {
            alive = mbar_wait_warp(empty0 + 8 * s, phase, err);
            if (!alive) break;
            if (elected) {
                arm_and_load_weights(i, s);
                tma_load_2d(b_base + s * B_BYTES, &map_x, (k_begin + i) * TC_BK, 0, full0 + 8 * s);
            }
            if (++s == STAGES) s = 0, phase ^= 1;
        }
    } else if (warp == 1) {
        const bool elected = elect_one();
        const unsigned long long da0 = umma_desc_sw128(a_base), db0 = umma_desc_sw128(b_base);
        bool alive = true;
        int s = 0, phase = 0;
        for (int i = 0; i < n_k; i++) {
            alive = mbar_wait_warp(full0 + 8 * s, phase, err);
            if (!alive) break;
            tc_fence_after();
            if (elected) {
                const unsigned long long da = da0 + s * (A_BYTES >> 4), db = db0 + s * (B_BYTES >> 4);
#pragma unroll
                for (int kk = 0; kk < TC_BK / 16; kk++) umma_bf16(tmem, da + 2 * kk, db + 2 * kk, IDESC, (i > 0 || kk > 0) ? 1u : 0u);
                umma_commit(empty0 + 8 * s);
            }
            if (++s == STAGES) s = 0, phase ^= 1;
        }
        if (elected) umma_commit(done_bar);
    } else {
        const int quad = warp & 3, row = quad * 32 + lane;
        asm volatile("griddepcontrol.wait;" ::: "memory");      // the workspace may still be read by an earlier kernel
        const bool ok = __all_sync(0xffffffffu, mbar_wait(done_bar, 0, err));
        tc_fence_after();
        const int ld = shrink ? v_ld : N;
        float* to = (shrink ? vs : base) + (size_t)blockIdx.z * T * ld + (shrink ? g0 * ADAPTER_GROUP : ra0) + row;
        if (ok)
#pragma unroll 1
            for (int c0 = 0; c0 < BN; c0 += 16) {
                if (c0 >= T) break;
                float v[16];
                tmem_ld16(tmem + ((unsigned)(quad * 32) << 16) + (unsigned)c0, v);
#pragma unroll
                for (int j = 0; j < 16; j++)
                    if (c0 + j < T && row < rows) to[(size_t)(c0 + j) * ld] = v[j];
            }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

__device__ __forceinline__ float ad_dot16(const float* w, const float* v, float acc) {
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const float4 f = reinterpret_cast<const float4*>(v)[q];
        acc = fmaf(f.x, w[4 * q], acc);
        acc = fmaf(f.y, w[4 * q + 1], acc);
        acc = fmaf(f.z, w[4 * q + 2], acc);
        acc = fmaf(f.w, w[4 * q + 3], acc);
    }
    return acc;
}

// TOK places of the plan's order by 128 threads, a column each; the loads of all places are in flight together.
template <int TOK, typename TOut>
__global__ void __launch_bounds__(AD_COLS)
adapter_join_kernel(const float* __restrict__ base, int splits, long long stride, int N, const bf16* __restrict__ b, const float* __restrict__ vs, int v_ld,
                    const float* __restrict__ scales, int R, const int4* __restrict__ places, int T, TOut* __restrict__ out) {
    __shared__ __align__(16) float v[TOK][ADAPTER_GROUP * ADAPTER_MAX_GROUPS];
    const int tid = threadIdx.x, col = blockIdx.x * AD_COLS + tid, p0 = blockIdx.y * TOK;
    int4 at[TOK];                                       // token, adapter, first group, groups
    int most = 0;
#pragma unroll
    for (int i = 0; i < TOK; i++) {                     // (the plan comes with a copy, not from a kernel)
        at[i] = p0 + i < T ? places[p0 + i] : make_int4(-1, -1, 0, 0);
        most = max(most, at[i].w);
    }
    // the second factors as well: the first groups' values come before the wait for the kernel that makes the slices
    const size_t ld = (size_t)(R / ADAPTER_GROUP) * N * ADAPTER_GROUP;
    uint4 head[TOK][2];
    if (col < N)
#pragma unroll
        for (int i = 0; i < TOK; i++)
            if (at[i].w > 0)
#pragma unroll
                for (int h = 0; h < 2; h++) head[i][h] = reinterpret_cast<const uint4*>(b + at[i].y * ld + (size_t)col * ADAPTER_GROUP)[h];
    pdl_grid_sync();
    float acc[TOK];
#pragma unroll
    for (int i = 0; i < TOK; i++) acc[i] = 0.f;
    if (col < N)
#pragma unroll 4
        for (int z = 0; z < splits; z++)
#pragma unroll
            for (int i = 0; i < TOK; i++)
                if (at[i].x >= 0) acc[i] += base[(size_t)z * stride + (size_t)at[i].x * N + col];
    if (most > 0) {
        // the places' rank values, a thread per rank of a place
        for (int q = tid; q < TOK * most * ADAPTER_GROUP; q += AD_COLS) {
            const int i = q / (most * ADAPTER_GROUP), rank = q - i * (most * ADAPTER_GROUP);
            int4 a = at[0];
#pragma unroll
            for (int e = 1; e < TOK; e++)
                if (i == e) a = at[e];
            if (rank < a.w * ADAPTER_GROUP) {
                const float* from = vs + (size_t)a.x * v_ld + a.z * ADAPTER_GROUP + rank;
                const float s = scales[a.y];
                float t = 0.f;
#pragma unroll 4
                for (int z = 0; z < splits; z++) t += from[(size_t)z * T * v_ld];
                v[i][rank] = s * t;
            }
        }
        __syncthreads();
        if (col < N)
            for (int g = 0; g < most; g++) {
                const bf16* next = b + ((size_t)(g + 1) * N + col) * ADAPTER_GROUP;
#pragma unroll
                for (int i = 0; i < TOK; i++)
                    if (g < at[i].w) {
                        float w[ADAPTER_GROUP];
                        load8(reinterpret_cast<const bf16*>(&head[i][0]), w);
                        load8(reinterpret_cast<const bf16*>(&head[i][1]), w + 8);
                        acc[i] = ad_dot16(w, &v[i][g * ADAPTER_GROUP], acc[i]);
                    }
#pragma unroll
                for (int i = 0; i < TOK; i++)
                    if (g + 1 < at[i].w)
#pragma unroll
                        for (int h = 0; h < 2; h++) head[i][h] = reinterpret_cast<const uint4*>(next + at[i].y * ld)[h];
            }
    }
    if (col < N)
#pragma unroll
        for (int i = 0; i < TOK; i++)
            if (at[i].x >= 0) out[(size_t)at[i].x * N + col] = from_f32<TOut>(acc[i]);
}

// How the rows form cuts K: as many slices as bring about two blocks to an SM, each at least 8 pieces of 64 wide, at most 8 slices (their reader pays for every one).
struct AdRows { int base_tiles, shrink_tiles, k_iters, per, splits; };
static AdRows ad_rows(int T, int N, int K, int groups) {
    AdRows r;
    r.base_tiles = ad_div(N, TC_BM);
    r.shrink_tiles = ad_div(groups, TC_BM / ADAPTER_GROUP);
    r.k_iters = ad_div(K, TC_BK);
    int s = 2 * illm_sm_count() / (r.base_tiles + r.shrink_tiles);
    s = s > r.k_iters / 8 ? r.k_iters / 8 : s;
    s = s > 8 ? 8 : s;
    s = s < 1 ? 1 : s;
    r.per = ad_div(r.k_iters, s);
    r.splits = ad_div(r.k_iters, r.per);
    return r;
}

template <int BN>
static int ad_launch_rows(const CUtensorMap& mw, const CUtensorMap& ma, const CUtensorMap& mx, float* base, float* vs, int v_ld, int T, int N, int R,
                          const AdRows& r, const AdPlan& plan, int early, int* err, cudaStream_t s) {
    const int stage = (TC_BM + BN) * TC_BK * 2;
    const int blocks = (r.base_tiles + r.shrink_tiles) * r.splits, sms = illm_sm_count();
    const int resident = blocks > 2 * sms ? 3 : (blocks > sms ? 2 : 1);
    int stages = (227 * 1024 / resident - 2560) / stage;
    stages = stages > AD_ROWS_MAX_STAGES ? AD_ROWS_MAX_STAGES : (stages < 2 ? 2 : stages);
    if (stages > r.per) stages = r.per < 2 ? 2 : r.per;
    const size_t smem = (size_t)stages * stage + 1024;
    auto kern = adapter_rows_kernel<BN>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    illm_launch(kern, dim3(r.base_tiles + r.shrink_tiles, 1, r.splits), dim3(TC_THREADS), smem, s, mw, ma, mx, base, vs, v_ld, T, N, R, r.base_tiles, plan,
                r.k_iters, r.per, stages, early, err);
    return illm_launch_status();
}

template <typename TOut>
static int ad_rows_form(const void* x, const void* w, int T, int N, int K, const void* a, const void* b, const float* scales, int count, int R,
                        const AdapterPlanSizes& sz, const int* plan_dev, TOut* out, char* ws, int early, int* err, cudaStream_t s) {
    const AdPlan plan = ad_plan(plan_dev, sz);
    const AdRows r = ad_rows(T, N, K, sz.groups);
    const int v_ld = sz.groups * ADAPTER_GROUP, bn = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : 128;
    float *vs = (float*)ws, *base = (float*)(ws + ad_round((long long)r.splits * T * v_ld * 4));
    CUtensorMap mw, ma, mx;
    int rc;
    if ((rc = ad_make_map(&mw, w, N, K, TC_BM)) || (rc = ad_make_map(&ma, a, (long long)count * R, K, ADAPTER_GROUP)) || (rc = ad_make_map(&mx, x, T, K, bn)))
        return rc;
    switch (bn) {
        case 16: rc = ad_launch_rows<16>(mw, ma, mx, base, vs, v_ld, T, N, R, r, plan, early, err, s); break;
        case 32: rc = ad_launch_rows<32>(mw, ma, mx, base, vs, v_ld, T, N, R, r, plan, early, err, s); break;
        case 64: rc = ad_launch_rows<64>(mw, ma, mx, base, vs, v_ld, T, N, R, r, plan, early, err, s); break;
        default: rc = ad_launch_rows<128>(mw, ma, mx, base, vs, v_ld, T, N, R, r, plan, early, err, s);
    }
    if (rc) return rc;
    auto join = [&](auto kern, int tok) {
        illm_launch(kern, dim3(ad_div(N, AD_COLS), ad_div(T, tok)), dim3(AD_COLS), 0, s, (const float*)base, r.splits, (long long)T * N, N, (const bf16*)b,
                    (const float*)vs, v_ld, scales, R, plan.places, T, out);
    };
    // A place to a block while that makes no more than some 11 blocks to an SM, else four.  One and four, us, L2 flushed, 4096 x N: 32
    // tokens of 4096 with 8 adapters of rank 64 19.0 and 20.8; of 6144 (10.4 blocks) with 32 of rank 16 20.6 and 20.7, of rank 64 28.5
    // and 30.3; 64 tokens of 3584 (12.1 blocks) with 64 of rank 16 20.8 and 18.9, of rank 64 31.8 and 31.8; of 4096 (13.8) 22.9 and 20.7,
    // 33.4 and 33.2; of 5120 25.0 and 22.8, 36.6 and 37.1.  (Mixed ranks fill four places unevenly: 64 tokens with 48 adapters of 11008 x
    // 4096 43.6 both ways, with the host between calls 31.4 and 33.2; far beyond the border they gain by one: of 4096 x 8192 37.5 and 40.3.)
    if (T * ad_div(N, AD_COLS) < 11 * illm_sm_count()) join(adapter_join_kernel<1, TOut>, 1);
    else join(adapter_join_kernel<4, TOut>, 4);
    return illm_launch_status();
}

// Where both forms can run, tiles are the faster one from 65 tokens on, and for wide products from 33 (rows form and tiles, us: 80
// tokens, 8 adapters of rank 64 beside 4096 x 4096 27.6 and 20.9, one of rank 16 beside 4096 x 12288 30.9 and 26.4; 64 tokens, 8 of
// rank 64 beside 11008 x 4096 30.5 and 36.0, beside 4096 x 12288 41.8 and 31.2; 32 with one beside 4096 x 22016 38.3 and 41.3).  With an adapter to every
// token they are not: 80 tokens with 64 of rank 16 beside 4096 x 4096 16.5 and 27.5.
static bool ad_tiled(int T, int slots, int N) { return adapter_tiled(T, slots) && (T > 64 || N > 64 * illm_sm_count()); }

// Bytes of workspace that illm_linear_adapters needs.
extern "C" long long illm_linear_adapters_ws(int dtype, int T, int N, int K, int R, int slots, int groups, int chunks) {
    if (dtype == ILLM_BF16 && !ad_tiled(T, slots, N)) {
        const long long splits = ad_rows(T, N, K, groups).splits;
        return ad_round(splits * T * groups * ADAPTER_GROUP * 4) + splits * T * N * 4;
    }
    return 256 + (dtype == ILLM_BF16 ? ad_prompt_ws(T, N, K, chunks) : (long long)T * R * 4);
}

static int ad_float32(const float* x, const float* w, int T, int N, int K, const float* a, const float* b, const float* scales, int R,
                      const AdapterPlanSizes& sz, const int* plan_dev, float* out, float* v, int early, int* err, cudaStream_t s) {
    const AdPlan plan = ad_plan(plan_dev, sz);
    const int rc = illm_gemm_f32_nt_ex(x, w, out, T, N, K, K, K, N, early, err, s);
    if (rc != 0) return rc;
    if (sz.slots == 0) return 0;
    const bool wide = K % 4 == 0 && !(((uintptr_t)x | (uintptr_t)a) & 15);
    auto shrink = wide ? adapter_shrink_kernel<4> : adapter_shrink_kernel<1>;
    illm_launch(shrink, dim3(ad_div(T, AD_SHRINK), R / ADAPTER_GROUP), dim3(256), 0, s, x, K, a, scales, R, plan.places, T, v);
    illm_launch(adapter_expand_kernel, dim3(ad_div(N, AD_COLS), ad_div(T, AD_TOKENS)), dim3(AD_COLS), 0, s, N, b, (const float*)v, R, plan.places, T, out);
    return illm_launch_status();
}

// out [T, N] = x W^T + the tokens' adapters.  dtype: of x, W, A and B; out_dtype float32 or that.  plan: the device array laid
// out by adapter_plan_layout({T, slots, groups, chunks}).  ws: illm_linear_adapters_ws bytes, 256-byte aligned.  early: no kernel ahead in
// the stream makes W, A or B, so that they may be read before the wait for it.
extern "C" int illm_linear_adapters(const void* x, const void* w, int dtype, int T, int N, int K, const void* a, const void* b, const float* scales,
                                    int count, int R, const int* plan, int slots, int groups, int chunks, void* out, int out_dtype, void* ws, int early,
                                    int* err, void* stream) {
    if (T <= 0 || N <= 0) return 0;
    if (K <= 0 || count <= 0 || R <= 0 || R % ADAPTER_GROUP || R > ADAPTER_GROUP * ADAPTER_MAX_GROUPS || slots < 0 || groups < 0 || chunks < 0 || !ws || !plan ||
        T > 65535 * AD_TOKENS || (long long)count * R * (N / ADAPTER_GROUP + 1) >= (1ll << 31) || (long long)count * R >= (1ll << 31))
        return ILLM_ERR_BAD_ARG;        // (rows of the factors are counted in 32 bits)
    if (dtype == ILLM_BF16 && ((K & 7) || ((uintptr_t)x & 15) || ((uintptr_t)w & 15) || ((uintptr_t)a & 15) || ((uintptr_t)b & 15))) return ILLM_ERR_BAD_ARG;
    const AdapterPlanSizes sz{T, slots, groups, chunks};
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == ILLM_F32 && out_dtype == ILLM_F32)
        return ad_float32((const float*)x, (const float*)w, T, N, K, (const float*)a, (const float*)b, scales, R, sz, plan, (float*)out, (float*)ws, early, err, s);
    if (dtype != ILLM_BF16 || (out_dtype != ILLM_BF16 && out_dtype != ILLM_F32)) return ILLM_ERR_BAD_ARG;
    if (ad_tiled(T, slots, N))
        return ad_prompt_form(x, w, T, N, K, a, b, scales, count, R, ad_plan(plan, sz), chunks, out, out_dtype, (char*)ws, err, s);
    if (out_dtype == ILLM_BF16) return ad_rows_form<bf16>(x, w, T, N, K, a, b, scales, count, R, sz, plan, (bf16*)out, (char*)ws, early, err, s);
    return ad_rows_form<float>(x, w, T, N, K, a, b, scales, count, R, sz, plan, (float*)out, (char*)ws, early, err, s);
}
