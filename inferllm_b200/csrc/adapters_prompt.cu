// Low-rank adapters beside a shared projection, for prompts in bfloat16: the adapters are a longer K.
//   y[t] = [x[t], v[t]] . [W, B]^T,   v[t] = s_a x[t] A_a^T
// For a tile of 256 tokens the further columns are the rank groups (16 ranks each) of the adapters that the tile's tokens name, four
// groups to a chunk of 64 columns; a token's v is zero in the groups of other adapters.  A prompt's tile names one or two
// adapters: one chunk behind the K / 64 pieces of the shared product, in the same accumulators, rounded once with it.
//
// adapter_values_kernel makes the chunks of v: 128 tokens by 64 ranks per cluster, tcgen05 (tokens on the lanes, four TMA boxes of
// 16 rows of A, or one of 64, as the MMA's N), the cluster's blocks share K and add up over distributed shared memory in the order of
// their ranks; scaled in float32, rounded to bfloat16 (the operand type of the product that follows; 2^-8 of a term that
// is itself a correction), zero where the token's adapter is another one.  Its bound is reading x once, from L2 behind the first chunk.
//
// adapter_pair_kernel is the product on pairs of SMs (tiles of 256 tokens by 96 to 256 outputs, cta_group::2, as gemm_tc2.cu: two
// blocks hold 128 token rows and half the weight rows each, persistent over the tiles, two accumulators in tensor memory).  A chunk
// is one more stage of its ring: 128 rows of v (128-byte swizzle) and four boxes of [half the outputs x 16 ranks] of B (32-byte
// swizzle, laid out so that a K step of 16 is one rank group of any adapter).  Few tiles: narrower ones, or slices of K, whose
// float32 sums a last kernel adds up (ap_shape).  It starts while the first kernel still runs: that one lets it go only when its own
// wait for the tokens' rows is over, so the shared product may be read at once, and only the chunks wait.
// Measured on one B200: 2,048 tokens of 4096 x 4096 with 12 adapters of mixed ranks 62 us (1,110 TFLOP/s, the product alone 51 to
// 55), 4,096 of 4096 x 22016 with rank 64 569 us (1,320 TFLOP/s, 94 % of what the library's product keeps up), 200 of
// 4096 x 6144 20.2 us, of which reading the weight takes 7.7.  Bound: the tensor cores from about 1,000 tokens on, below that
// the latency of launching, filling and draining two dependent kernels.
#include "adapters.cuh"
#include "kernels.h"
#include "tc_pair.cuh"

#define AP_VALUE_STAGES 8
#define AP_VALUE_THREADS 256
#define AP_COLS (ADAPTER_CHUNK * ADAPTER_GROUP)        // columns of a chunk
#define AP_PITCH (AP_COLS + 4)      // floats: rows start on 16 bytes, and 8 neighbouring ones in different banks
#define AP_OUT_PITCH 33
#define AP_THREADS 224             // of the product: two warps fetch, one multiplies, four finish

__device__ __forceinline__ float4 ap_load_remote(const float* local, unsigned rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(map_to_cta(tc_smem_u32(local), rank)) : "memory");
    return v;
}

// grid: cluster blocks of a half tile, halves, chunks, in this order along x
template <int AP_ITEMS>
__global__ void __launch_bounds__(AP_VALUE_THREADS)
adapter_values_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_a4, const float* __restrict__ scales, int R, int T,
                      int C, int k_iters_total, int STAGES, const AdPlan plan, bf16* __restrict__ v, int* __restrict__ err) {
    constexpr unsigned A_BYTES = TC_BM * TC_BK * 2, B_BYTES = AP_COLS * TC_BK * 2, BOX_BYTES = ADAPTER_GROUP * TC_BK * 2;
    static_assert((A_BYTES + B_BYTES) * 2 >= TC_BM * AP_PITCH * 4, "two stages hold the sums");
    constexpr unsigned IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(AP_COLS >> 3) << 17) | ((unsigned)(TC_BM >> 4) << 24);
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * AP_VALUE_STAGES + 1];
    __shared__ unsigned tmem_holder;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int chunk = (int)blockIdx.x / (2 * C), half = (int)blockIdx.x / C & 1;
    const unsigned rank = cluster_ctarank();
    const int n_chunks = plan.counts[2], t0 = plan.chunk_tile[chunk] * ADAPTER_TILE + half * TC_BM;
    const int4 groups = *reinterpret_cast<const int4*>(plan.chunk_groups + chunk * ADAPTER_CHUNK);
    if (chunk >= n_chunks) {                            // the grid is sized for more chunks than there are (all blocks of the cluster leave)
        asm volatile("griddepcontrol.wait;" ::: "memory");      // (the product relies on this kernel's wait)
        return;
    }

    const unsigned a_base = (tc_smem_u32(smem_raw) + 1023u) & ~1023u, b_base = a_base + STAGES * A_BYTES;
    float* partial = reinterpret_cast<float*>(smem_raw + (a_base - tc_smem_u32(smem_raw)));     // [128][AP_PITCH] over the ring, when it is done
    const unsigned full0 = tc_smem_u32(&bars[0]), empty0 = tc_smem_u32(&bars[AP_VALUE_STAGES]), done_bar = tc_smem_u32(&bars[2 * AP_VALUE_STAGES]);
    const int per = (k_iters_total + C - 1) / C, k_begin = (int)rank * per, n_k = max(0, min(per, k_iters_total - k_begin));

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(full0 + 8 * s, 2);
            mbar_init(empty0 + 8 * s, 1);
        }
        mbar_init(done_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(&tmem_holder)), "r"((unsigned)AP_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_holder;

    if (warp <= 1) {
        // (the warps stay together around what one lane issues: what every lane agrees on then lies in uniform registers)
        const bool elected = elect_one();
        // warp 0 fetches the tokens' rows (and hears from the MMAs when a stage is free), warp 1 the adapters'; a stage is full when
        // both have arrived
        int row[ADAPTER_CHUNK], boxes = 0;
        bool joined = true;                             // the four groups lie one behind another: one box instead of four
#pragma unroll
        for (int j = 0; j < ADAPTER_CHUNK; j++) {
            const int g = j == 0 ? groups.x : j == 1 ? groups.y : j == 2 ? groups.z : groups.w;
            row[j] = g < 0 ? -1 : (g / ADAPTER_MAX_GROUPS) * R + (g % ADAPTER_MAX_GROUPS) * ADAPTER_GROUP;
            boxes += g >= 0;
            joined = joined && row[j] == row[0] + j * ADAPTER_GROUP && g >= 0;
        }
        asm volatile("griddepcontrol.wait;" ::: "memory");
        // only now may the product begin: it reads the tokens' rows without a wait of its own
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        bool alive = true;
        int s = 0, phase = 1;
        for (int i = 0; i < n_k; i++) {
            if (i >= STAGES) alive = mbar_wait_warp(empty0 + 8 * s, phase, err);
            if (!alive) break;
            const int kx = (k_begin + i) * TC_BK;
            if (!elected) {
            } else if (warp == 0) {
                mbar_expect_tx(full0 + 8 * s, A_BYTES);
                tma_load_2d(a_base + s * A_BYTES, &map_x, kx, t0, full0 + 8 * s);
            } else {
                mbar_expect_tx(full0 + 8 * s, boxes * BOX_BYTES);
                if (joined) {
                    tma_load_2d(b_base + s * B_BYTES, &map_a4, kx, row[0], full0 + 8 * s);
                } else {
#pragma unroll
                    for (int j = 0; j < ADAPTER_CHUNK; j++)
                        if (row[j] >= 0) tma_load_2d(b_base + s * B_BYTES + j * BOX_BYTES, &map_a, kx, row[j], full0 + 8 * s);
                }
            }
            if (++s == STAGES) s = 0, phase ^= 1;
        }
    } else if (warp == 2) {
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
    }
    // each block finishes its share of the rows, four columns to a thread: what it needs for that, while the products run
    const int rows = TC_BM / C, items = rows * (AP_COLS / 4);
    float factor[AP_ITEMS];
    asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll
    for (int q = 0; q < AP_ITEMS; q++) {
        const int i = threadIdx.x + q * AP_VALUE_THREADS, t = t0 + (int)rank * rows + i / (AP_COLS / 4);
        const int j = i % (AP_COLS / 4) / (ADAPTER_GROUP / 4), g = j == 0 ? groups.x : j == 1 ? groups.y : j == 2 ? groups.z : groups.w, ad = i < items && t < T ? plan.token_adapter[t] : -1;
        factor[q] = g >= 0 && g / ADAPTER_MAX_GROUPS == ad ? scales[ad] : NAN;        // NaN: the token's adapter is another one
    }
    __syncwarp();
    if (warp >= AP_VALUE_THREADS / 32 - 4) {
        const int quad = warp & 3, r = quad * 32 + lane;
        const bool ok = __all_sync(0xffffffffu, mbar_wait(done_bar, 0, err));
        tc_fence_after();
#pragma unroll
        for (int c0 = 0; c0 < AP_COLS; c0 += 16) {
            float f[16];
            if (ok && n_k > 0) tmem_ld16(tmem + ((unsigned)(quad * 32) << 16) + (unsigned)c0, f);
#pragma unroll
            for (int j = 0; j < 16; j++) f[j] = ok && n_k > 0 ? f[j] : 0.f;
            store8(partial + r * AP_PITCH + c0, f);
            store8(partial + r * AP_PITCH + c0 + 8, f + 8);
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                 // every block's sums are there
    if (warp == 2) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((unsigned)AP_COLS) : "memory");
    }
#pragma unroll
    for (int q = 0; q < AP_ITEMS; q++) {
        const int i = threadIdx.x + q * AP_VALUE_THREADS, r = (int)rank * rows + i / (AP_COLS / 4), c = i % (AP_COLS / 4) * 4;
        if (i >= items) break;
        float f[4] = {0.f, 0.f, 0.f, 0.f};
        if (factor[q] == factor[q]) {
            float4 p[8];
#pragma unroll
            for (int b = 0; b < 8; b++) p[b] = b < C ? ap_load_remote(&partial[r * AP_PITCH + c], b) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int b = 0; b < 8; b++) f[0] += p[b].x, f[1] += p[b].y, f[2] += p[b].z, f[3] += p[b].w;
#pragma unroll
            for (int j = 0; j < 4; j++) f[j] *= factor[q];
        }
        __nv_bfloat162 o[2] = {__floats2bfloat162_rn(f[0], f[1]), __floats2bfloat162_rn(f[2], f[3])};
        *reinterpret_cast<uint2*>(v + ((size_t)chunk * ADAPTER_TILE + half * TC_BM + r) * AP_COLS + c) = *reinterpret_cast<uint2*>(o);
    }
    cluster_sync_all();                                 // no block leaves while another may still read its sums
}

// Descriptor of a K-major tile whose rows are 32 bytes, 32-byte swizzled: 8-row groups 256 bytes apart.
__device__ __forceinline__ unsigned long long umma_desc_sw32(unsigned smem_addr) {
    return (unsigned long long)((smem_addr & 0x3FFFF) >> 4) | (1ull << 16) | ((unsigned long long)(256 >> 4) << 32) | (1ull << 46) | (6ull << 61);
}

// C = x . W^T + the chunks.  splits > 1: C is float32 [splits, T, N], slice z the z-th run of K pieces, the last with the chunks.
// (Tiles of 512 outputs, which need 48 KB instead of 64 for the same work but cannot hide their epilogue, were 3 to 15 % slower.)
// Even, so that a stage is always the same warp's to fill: a wait by parity holds only for one that has seen the phase before.
template <int BN> constexpr int ap_stages() { return 192 * 1024 / ((TC_BM + BN / 2) * TC_BK * 2) / 2 * 2; }
template <int BN, typename TOut>
__global__ void __launch_bounds__(AP_THREADS)
adapter_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ CUtensorMap map_b, TOut* __restrict__ C, int T, int N, int R, int k_iters_total, int splits, const AdPlan plan,
                    int chunked, int* __restrict__ err) {
    constexpr int STAGES = ap_stages<BN>(), HALF = BN / 2;
    constexpr unsigned A_BYTES = TC_BM * TC_BK * 2, B_BYTES = HALF * TC_BK * 2, BOX_BYTES = HALF * ADAPTER_GROUP * 2;
    constexpr unsigned TMEM_COLS = 512;
    constexpr unsigned IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(BN >> 3) << 17) | ((unsigned)(256 >> 4) << 24);
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const unsigned base = tc_smem_u32(smem_raw);
    const unsigned a_base = base, b_base = a_base + STAGES * A_BYTES;
    const unsigned bars = b_base + STAGES * B_BYTES;
    const unsigned full0 = bars, empty0 = bars + 8 * STAGES;
    const unsigned acc_full0 = bars + 16 * STAGES, acc_empty0 = acc_full0 + 16;
    unsigned* tmem_holder = reinterpret_cast<unsigned*>(smem_raw + (bars - base) + 16 * STAGES + 32);
    float* stage_out = reinterpret_cast<float*>(smem_raw + (bars - base) + 16 * STAGES + 48);       // [4][32][AP_OUT_PITCH], only for odd N

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const int n_m = (T + 255) / 256, n_tiles = n_m * ((N + BN - 1) / BN), n_items = n_tiles * splits;
    const int per = (k_iters_total + splits - 1) / splits;

    if ((base & 1023u) != 0) {          // no static shared memory is declared: cannot happen; never run misaligned
        if (threadIdx.x == 0) atomicExch(err, TC_ERR_MISALIGNED_SMEM);
        return;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(acc_full0 + 8 * b, 1);
            mbar_init(acc_empty0 + 8 * b, 8);      // four epilogue warps in each of the two blocks
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(tmem_holder)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                 // the peer's barriers exist before anything arrives on them
    tc_fence_after();
    const unsigned tmem = *tmem_holder;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // item -> its tile, its run of K pieces and its chunks
    auto item = [&](int i, int& m, int& n, int& k0, int& k1, int& c0, int& c1) {
        const int z = i / n_tiles, t = i - z * n_tiles;
        m = t % n_m, n = t / n_m;
        k0 = z * per, k1 = min(k_iters_total, k0 + per);
        c0 = c1 = 0;
        if (chunked && z == splits - 1) c0 = plan.tile_chunk[m], c1 = plan.tile_chunk[m + 1];
    };
    if (warp == 0 || warp == 6) {
        // two warps that fetch, each every other piece (one of them takes about 0.22 us for a piece's wait, its announcement and its
        // two loads; a warp stays together around what one lane issues, which costs it a third less than a lane by itself)
        const bool elected = elect_one();
        const int turn = warp == 6;
        bool alive = true, waited = false;
        int s = turn, phase = 1, it = 0;
        const unsigned full_leader = map_to_cta(full0, 0);      // block 0 counts the bytes of both
        if (!chunked) asm volatile("griddepcontrol.wait;" ::: "memory");       // no kernel of ours has waited for the tokens' rows
        for (int i = pair; i < n_items && alive; i += n_pairs) {
            int m, n, k0, k1, c0, c1;
            item(i, m, n, k0, k1, c0, c1);
            const int ra0 = m * 256 + (int)rank * 128, rb0 = n * BN + (int)rank * HALF, end = k1 + (c1 - c0);
            // `it` counts the pieces of all items
            for (int k = k0 + ((it ^ turn) & 1); k < end; k += 2) {
                if (it + (k - k0) >= STAGES) alive = mbar_wait_warp(empty0 + 8 * s, phase, err);
                if (!alive) break;
                const unsigned a_s = a_base + s * A_BYTES, b_s = b_base + s * B_BYTES, full = full_leader + 8 * s;
                if (k < k1) {
                    if (elected) {
                        if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * (A_BYTES + B_BYTES));
                        tma_load_2d_pair(b_s, &map_w, k * TC_BK, rb0, full);
                        tma_load_2d_pair(a_s, &map_x, k * TC_BK, ra0, full);
                    }
                } else {
                    const int c = c0 + (k - k1);
                    int g[ADAPTER_CHUNK], boxes = 0;
#pragma unroll
                    for (int j = 0; j < ADAPTER_CHUNK; j++) {
                        g[j] = plan.chunk_groups[c * ADAPTER_CHUNK + j];
                        boxes += g[j] >= 0;
                    }
                    if (!waited) {
                        asm volatile("griddepcontrol.wait;" ::: "memory");     // the values are there
                        waited = true;
                    }
                    if (elected) {
                        if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * (A_BYTES + boxes * BOX_BYTES));
                        tma_load_2d_pair(a_s, &map_v, 0, c * ADAPTER_TILE + (int)rank * 128, full);
#pragma unroll
                        for (int j = 0; j < ADAPTER_CHUNK; j++)
                            if (g[j] >= 0) {
                                const int row = ((g[j] / ADAPTER_MAX_GROUPS) * (R / ADAPTER_GROUP) + g[j] % ADAPTER_MAX_GROUPS) * N + rb0;
                                tma_load_2d_pair(b_s + j * BOX_BYTES, &map_b, 0, row, full);
                            }
                    }
                }
                s += 2;
                if (s >= STAGES) s -= STAGES, phase ^= 1;
            }
            it += end - k0;
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const bool elected = elect_one();
            bool alive = true;
            int s = 0, phase = 0, ti = 0;
            // descriptors of the first stage; 16 bytes are one unit of their address
            const unsigned long long da0 = umma_desc_sw128(a_base), db0 = umma_desc_sw128(b_base);
            for (int i = pair; i < n_items && alive; i += n_pairs, ti++) {
                int m, n, k0, k1, c0, c1;
                item(i, m, n, k0, k1, c0, c1);
                const int buf = ti & 1;
                const unsigned d = tmem + buf * 256;
                if (ti >= 2) alive = mbar_wait_warp(acc_empty0 + 8 * buf, ((ti >> 1) - 1) & 1, err);
                tc_fence_after();
                // (one thread issues every MMA of the pair: its loop over K holds nothing but waits and MMAs, and the chunks have
                // their own; with a choice between the two inside, 4,096 tokens of 4096 x 22016 took 610 us instead of 479.  Two pieces
                // to a round of it: 200 tokens of 2048 x 2048 9.6 us instead of 11.1, of 4096 x 6144 18.0 instead of 18.7)
                auto multiply = [&](int stage, unsigned accumulate) {
                    const unsigned long long da = da0 + stage * (A_BYTES >> 4), db = db0 + stage * (B_BYTES >> 4);
#pragma unroll
                    for (int kk = 0; kk < TC_BK / 16; kk++) umma_bf16_pair(d, da + 2 * kk, db + 2 * kk, IDESC, kk > 0 ? 1u : accumulate);
                    umma_commit_pair(empty0 + 8 * stage);
                };
                int k = k0;
                for (; k + 1 < k1 && alive; k += 2) {
                    const int s2 = s + 1 == STAGES ? 0 : s + 1, phase2 = s2 == 0 ? phase ^ 1 : phase;
                    alive = __all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, phase, err) && mbar_wait(full0 + 8 * s2, phase2, err));
                    if (!alive) break;
                    tc_fence_after();
                    if (elected) {
                        multiply(s, k > k0 ? 1u : 0u);
                        multiply(s2, 1u);
                    }
                    s = s2 + 1 == STAGES ? 0 : s2 + 1;
                    phase = s == 0 ? phase2 ^ 1 : phase2;
                }
                if (k < k1 && alive) {
                    alive = mbar_wait_warp(full0 + 8 * s, phase, err);
                    tc_fence_after();
                    if (elected && alive) multiply(s, k > k0 ? 1u : 0u);
                    if (++s == STAGES) s = 0, phase ^= 1;
                }
                for (int c = c0; c < c1 && alive; c++) {
                    alive = mbar_wait_warp(full0 + 8 * s, phase, err);
                    if (!alive) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int kk = 0; kk < ADAPTER_CHUNK; kk++)
                        if (elected && plan.chunk_groups[c * ADAPTER_CHUNK + kk] >= 0)
                            umma_bf16_pair(d, da0 + s * (A_BYTES >> 4) + 2 * kk, umma_desc_sw32(b_base + s * B_BYTES + kk * BOX_BYTES), IDESC, 1u);
                    if (elected) umma_commit_pair(empty0 + 8 * s);
                    if (++s == STAGES) s = 0, phase ^= 1;
                }
                if (elected) umma_commit_pair(acc_full0 + 8 * buf);
            }
        }
    } else {
        const int quad = warp & 3;
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const unsigned acc_empty_leader = map_to_cta(acc_empty0, 0);
        bool alive = true;
        int ti = 0;
        for (int i = pair; i < n_items && alive; i += n_pairs, ti++) {
            int m, n, k0, k1, c0, c1;
            item(i, m, n, k0, k1, c0, c1);
            const int buf = ti & 1, ra = m * 256 + (int)rank * 128 + quad * 32 + lane, rb0 = n * BN;
            TOut* Cz = C + (size_t)(i / n_tiles) * T * N;
            // lanes leave the polling loop one by one: together again before the warp-wide tcgen05.ld
            alive = __all_sync(0xffffffffu, mbar_wait(acc_full0 + 8 * buf, (ti >> 1) & 1, err));
            if (!alive) break;
            tc_fence_after();
            const unsigned tbase = tmem + ((unsigned)(quad * 32) << 16) + (unsigned)(buf * 256);
            if ((N & 7) == 0) {
#pragma unroll 1
                for (int c = 0; c < BN; c += 16) {
                    if (rb0 + c >= N) break;
                    float v[16];
                    tmem_ld16(tbase + c, v);
                    if (ra < T) {
                        TOut* dst = Cz + (size_t)ra * N + rb0 + c;
                        store8(dst, v);
                        if (rb0 + c + 8 < N) store8(dst + 8, v + 8);
                    }
                }
            } else {
                // rows that start anywhere: 32 of them by 32 columns through shared memory, so that a warp stores a row's neighbours
                // together (element by element, a row to a thread, 260 tokens of 2048 x 32001 took 205 us)
                float* mine = stage_out + (warp - 2) * 32 * AP_OUT_PITCH;
                const int rows = min(32, T - (ra - lane));
#pragma unroll 1
                for (int c = 0; c < BN; c += 32) {
                    if (rb0 + c >= N) break;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float v[16];
                        tmem_ld16(tbase + c + 16 * h, v);
#pragma unroll
                        for (int j = 0; j < 16; j++) mine[lane * AP_OUT_PITCH + 16 * h + j] = v[j];
                    }
                    __syncwarp();
                    if (rb0 + c + lane < N) {
                        TOut* dst = Cz + (size_t)(ra - lane) * N + rb0 + c + lane;
#pragma unroll 4
                        for (int q = 0; q < rows; q++) store_out<TOut>(dst + (size_t)q * N, mine[q * AP_OUT_PITCH + lane]);
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_empty_leader + 8 * buf);
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                 // neither block leaves while the other may still touch it
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// out[i] = the slices' sum in ascending order, four neighbours a thread
template <typename TOut> __global__ void __launch_bounds__(256) adapter_sum_kernel(const float* __restrict__ slices, int splits, long long n, TOut* __restrict__ out) {
    pdl_grid_sync();
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    float4 f[4];                                        // (at most 4 slices)
#pragma unroll
    for (int z = 0; z < 4; z++) f[z] = z < splits ? *reinterpret_cast<const float4*>(slices + z * n + i) : make_float4(0.f, 0.f, 0.f, 0.f);
    float a[4] = {f[0].x, f[0].y, f[0].z, f[0].w};
#pragma unroll
    for (int z = 1; z < 4; z++) a[0] += f[z].x, a[1] += f[z].y, a[2] += f[z].z, a[3] += f[z].w;
    AdColumns<4>::store(out + i, a);
}

// ---- host side

// How the shared product is cut: the width of its tiles, the slices of K and the blocks that share a chunk's values.
struct ApShape { int bn, splits, C; };

// Blocks that share a chunk's K: the product's pairs of SMs start at once where the kernel of the values leaves SMs free, and those
// that start behind it should be the ones that the last round of tiles would leave idle (2,048 tokens of 4096 x 4096: 57 us, 67
// with blocks everywhere), as long as a block's share of K is no longer than a tile's; else about two blocks to an SM.
static int ap_values_blocks(int items, int chunks, int k_iters, int splits) {
    const int most_pairs = illm_sm_count() / 2;
    const int idle = 2 * (items <= most_pairs ? most_pairs - items : (most_pairs - items % most_pairs) % most_pairs);
    auto share = [&](int room) {
        int c = 1;
        while (c < 8 && chunks * 2 * c * 2 <= room && k_iters >= 4 * c) c *= 2;
        return c;
    };
    const int c = share(idle);
    return chunks * 2 * c > idle || ad_div(k_iters, c) > ad_div(k_iters, splits) ? share(2 * illm_sm_count()) : c;
}

// The least of an estimate in us over widths of 96 to 256 and up to 4 slices.  A pair of SMs counts max(0.18, 0.045 + 0.0011 width) for
// a piece of 64 (the narrow ones are bound by the waits and the issue of the pieces; measured before the multiplying warp took two
// to a round, which leaves the order of the widths), the tiles come in rounds of as many as there are
// pairs; the values of the last chunk take 3 and 0.42 a piece, beside it or before it; slices cost their kernel, 2, and their bytes twice.
// Measured with 256 wide tiles (with slices where they do not fill the pairs) and with the choice: 200 tokens of 4096 x 6144 29.0
// and 18.7 us, 512 of 4096 x 4096 24.9 and 18.8, 1,000 of 4096 x 6144 47.2 and 42.3, 257 of 1024 x 1024 14.8 and 9.3.  Against the
// best of all widths and slices over 14 sizes of 150 to 2,048 tokens, replayed behind a flush of L2: up to 3 % more in 13 of them, 12 %
// (17.9 and 16.0 us) at 257 of 1024 x 1024.
static ApShape ap_shape(int T, int N, int K, int chunks) {
    const int k_iters = ad_div(K, TC_BK), pairs = illm_sm_count() / 2;
    ApShape best{256, 1, 1};
    float least = 0.f;
    for (int bn = 256; bn >= 96; bn -= 32)
        for (int want = 1; want <= 4; want++) {
            const int pieces = ad_div(k_iters, want), splits = ad_div(k_iters, pieces), items = ad_div(T, 256) * ad_div(N, bn) * splits;
            if (splits != want || (splits > 1 && (items > pairs || pieces < 8))) continue;
            const int C = chunks > 0 ? ap_values_blocks(items, chunks, k_iters, splits) : 1;
            const float piece = 0.045f + 0.001075f * bn, product = ad_div(items, pairs) * pieces * (piece < 0.18f ? 0.18f : piece);
            // (where they find no SM left free the product's blocks wait for theirs)
            const float values = chunks > 0 ? 3.f + 0.42f * ad_div(k_iters, C) : 0.f;
            const bool beside = chunks * 2 * C <= 2 * (pairs - items % pairs) % (2 * pairs);
            const float time = (!beside ? product + values : product < values ? values : product) + (splits > 1 ? 2.f + (float)splits * T * N * 1.6e-6f : 0.f);
            if (least == 0.f || time < least) least = time, best = ApShape{bn, splits, C};
        }
    return best;
}
long long ad_prompt_ws(int T, int N, int K, int chunks) {
    const int s = ap_shape(T, N, K, chunks).splits;
    return ad_round((long long)chunks * ADAPTER_TILE * AP_COLS * 2) + (s > 1 ? (long long)s * T * N * 4 : 0);
}

template <int BN, typename TOut>
static int ap_launch_pair(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mv, const CUtensorMap& mb, TOut* out, int T, int N, int R, int k_iters,
                          int splits, const AdPlan& plan, int chunked, int* err, cudaStream_t s) {
    const size_t smem = (size_t)ap_stages<BN>() * (TC_BM + BN / 2) * TC_BK * 2 + 16 * ap_stages<BN>() + 32 + 16 + ((N & 7) ? 4 * 32 * AP_OUT_PITCH * 4 : 0);
    auto kern = adapter_pair_kernel<BN, TOut>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    const int items = ad_div(T, 256) * ad_div(N, BN) * splits, most = illm_sm_count() / 2, pairs = items < most ? items : most;
    return illm_launch_cluster(kern, dim3(2 * pairs), dim3(AP_THREADS), 2, smem, s, mx, mw, mv, mb, out, T, N, R, k_iters, splits, plan, chunked, err);
}

template <typename TOut>
static int ap_launch(int bn, const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mv, const CUtensorMap& mb, TOut* out, int T, int N, int R, int k_iters,
                     int splits, const AdPlan& plan, int chunked, int* err, cudaStream_t s) {
    switch (bn) {
#define AP_CASE(W) case W: return ap_launch_pair<W>(mx, mw, mv, mb, out, T, N, R, k_iters, splits, plan, chunked, err, s);
        AP_CASE(96) AP_CASE(128) AP_CASE(160) AP_CASE(192) AP_CASE(224)
#undef AP_CASE
        default: return ap_launch_pair<256>(mx, mw, mv, mb, out, T, N, R, k_iters, splits, plan, chunked, err, s);
    }
}

int ad_prompt_form(const void* x, const void* w, int T, int N, int K, const void* a, const void* b, const float* scales, int count, int R,
                   const AdPlan& plan, int chunks, void* out, int out_dtype, char* ws, int* err, cudaStream_t s) {
    const ApShape shape = ap_shape(T, N, K, chunks);
    const int k_iters = ad_div(K, TC_BK), splits = shape.splits, bn = shape.bn, C = shape.C;
    bf16* v = (bf16*)ws;
    float* slices = (float*)(ws + ad_round((long long)chunks * ADAPTER_TILE * AP_COLS * 2));
    CUtensorMap mx, ma, ma4, mw, mv, mb;
    int rc;
    if ((rc = ad_make_map(&mx, x, T, K, TC_BM)) || (rc = ad_make_map(&mw, w, N, K, bn / 2))) return rc;
    mv = mb = mx;
    if (chunks > 0) {
        if ((rc = ad_make_map(&ma, a, (long long)count * R, K, ADAPTER_GROUP)) || (rc = ad_make_map(&ma4, a, (long long)count * R, K, AP_COLS)) ||
            (rc = ad_make_map(&mv, v, (long long)chunks * ADAPTER_TILE, AP_COLS, TC_BM)) ||
            (rc = ad_make_map(&mb, b, (long long)count * (R / ADAPTER_GROUP) * N, ADAPTER_GROUP, bn / 2, ADAPTER_GROUP, CU_TENSOR_MAP_SWIZZLE_32B)))
            return rc;
        // the ring holds a block's whole share of K where one block has an SM to itself
        const int per = ad_div(k_iters, C), most = chunks * 2 * C > illm_sm_count() ? 4 : AP_VALUE_STAGES, stages = per < 2 ? 2 : per < most ? per : most;
        const size_t smem = (size_t)stages * (TC_BM + AP_COLS) * TC_BK * 2 + 1024;
        // rows and columns that a thread finishes: 128 / C x 64 in fours, 256 threads
        auto kern = C == 8 ? adapter_values_kernel<1> : C == 4 ? adapter_values_kernel<2> : C == 2 ? adapter_values_kernel<4> : adapter_values_kernel<8>;
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        rc = illm_launch_cluster(kern, dim3((unsigned)C * 2 * chunks), dim3(AP_VALUE_THREADS), C, smem, s, mx, ma, ma4, scales, R, T, C, k_iters, stages, plan, v, err);
        if (rc) return rc;
    }
    if (splits > 1) {
        rc = ap_launch<float>(bn, mx, mw, mv, mb, slices, T, N, R, k_iters, splits, plan, chunks > 0, err, s);
        if (rc) return rc;
        const long long n = (long long)T * N;
        if (n % 4 || ((uintptr_t)out & 15)) return illm_splitk_reduce(slices, out, out_dtype, n, splits, s);
        const dim3 blocks((unsigned)((n / 4 + 255) / 256));
        if (out_dtype == ILLM_BF16) illm_launch(adapter_sum_kernel<bf16>, blocks, dim3(256), 0, s, (const float*)slices, splits, n, (bf16*)out);
        else illm_launch(adapter_sum_kernel<float>, blocks, dim3(256), 0, s, (const float*)slices, splits, n, (float*)out);
        return illm_launch_status();
    }
    if (out_dtype == ILLM_BF16) return ap_launch<bf16>(bn, mx, mw, mv, mb, (bf16*)out, T, N, R, k_iters, 1, plan, chunks > 0, err, s);
    return ap_launch<float>(bn, mx, mw, mv, mb, (float*)out, T, N, R, k_iters, 1, plan, chunks > 0, err, s);
}
