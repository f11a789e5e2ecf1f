// Attention of many queries over paged caches on the 5th-generation tensor cores where the rows of the products are (token, head)
// pairs that share a key/value head: prompts over rows of eight bits (kv_int8.cu), and the tokens of a step over a prefix that their
// sequences hold in common (eight bits or bfloat16), which is then read once for all of them.
//
//   o = sum_j p_j v_j,  p = softmax over the visible j of scale q . k_j       (src/kern/naive/naive.cpp:606-632, :531-553, :209-240, :664-691)
//
// A block has two tiles of 128 rows over the same keys and is alone on its SM.  Eight softmax warps (a thread is a row of a tile and a lane of
// tensor memory), a thread that issues the products, one that brings pages by TMA and, for eight bits, four warps that widen them:
// bytes from a ring of four raw stages become u - 128 in bfloat16, exactly, in the swizzled layout that the products read.  Widening
// costs about two instructions an element, which is why the tiles share it; two rows five apart (r and r XOR 5) go to a quarter of a warp, so that neither
// its loads nor its stores meet in a bank.  The rows' scales are factors of the scores and, the values', of the softmax weights.
// Tensor memory: the tiles' outputs, their scores of 64 keys, their weights (32 columns) and the first tile's queries, 512 columns at head size 128.
// With both operands in shared memory a product of 128 x 64 x 16 took about 95 clocks, as much again as one of twice the size whose rows come from
// tensor memory, and 256 rows were bound by that.  The scores of the next keys are made while the softmax works on the last ones; the output is rescaled
// only when a row's maximum has grown by more than 2^8.
// Rounded to bfloat16 are the softmax weights (times the value's scale) and the results; scores, sums and the running output are float32.  (Rows
// widened with their scales in them, and so rounded, put the results 0.006 of their norm off at scores of spread 2; like this it is 0.002.)
// One prompt of 4,096 tokens behind 2,001 of 32 heads of 128 takes 320 to 340 us (0.8 to 0.85 PFLOP/s): 57 % of the issue slots, the exponentials 44 % of their unit and the
// products 43 % of theirs; a prefix of 8,192 positions under 64 tokens of 32 / 8 heads 28.
// A key whose row reads back as NaN has its score NaN instead, so that it reaches the queries that see it and no others.
#include <cuda.h>
#include <math.h>

#include "attention_tc.cuh"
#include "paged_rows.cuh"
#include "tc_common.cuh"

#define TL_BM 128
#define TL_BN 64
#define TL_RAW 4                        // raw stages (eight bits)
#define TL_SOFTMAX 8                    // warps
#define TL_MMA_WARP 8                   // the first of two, one for each tile
#define TL_TMA_WARP 10
#define TL_WIDEN_WARP 11                // the first of four
#define TL_ERR_PAGE 8
#define TL_ORDERED 128                  // sequences that are put in order
#define TL_CLUSTER 4                    // parts of a prefix that join their shares: of clusters of eight such blocks only 15 find room, of four 33
#define TL_RESCALE_STEP 8.0f

// Which rows and keys: prompts (PREFIX false) or the tiles of a plan of common prefixes (attention_pages.cu).
struct TlWork {
    const int *cu_q, *seq_lens;         // prompts: [B + 1], [B]
    int span, tile_rows;                // tile_rows: rows of a block, 128 (its first tile alone) or 256
    const int4* tiles;                  // prefixes: members, positions, 0, 0
    const int *members, *token_seq;     // 256 / (nh / nkv) places for the members of each tile
    int slots, slot0;                   // shares of a (token, head) and the first of them that is the prefix's
    int cluster;                        // blocks (parts of a prefix) that join their shares
    float *part_acc, *part_ml;
};

template <int D, bool Q8> struct TlSizes {
    static constexpr int STAGES = Q8 ? 2 : 4, TILE = TL_BN * D * 2, Q_TILE = TL_BM * D * 2;
    static constexpr int RAW_TILE = TL_BN * D, RAW = Q8 ? TL_RAW : 0, SCALES = 2 * TL_BN * 4;
    static constexpr int SMEM = 2 * Q_TILE + STAGES * 2 * TILE + RAW * (2 * RAW_TILE + 2 * SCALES) + 512;
    static constexpr int THREADS = (Q8 ? 15 : 11) * 32;
};

namespace {

__device__ __forceinline__ void tl_arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void tl_store16(unsigned at, unsigned a, unsigned b, unsigned c, unsigned d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// sixteen bytes as u - 128 in bfloat16, exactly: a byte below 0x4b0000 is 2^23 + u in float32, and the difference has at most seven bits, which
// are the upper half of its word
__device__ __forceinline__ void tl_widen(const unsigned (&w)[4], unsigned (&out)[8]) {
    const unsigned long long bias = f2_pack(-8388736.f, -8388736.f);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const unsigned lo = __byte_perm(w[i], 0x4b000000u, h ? 0x7652 : 0x7650), hi = __byte_perm(w[i], 0x4b000000u, h ? 0x7653 : 0x7651);
            float a, b;
            f2_unpack(f2_add(f2_pack(__uint_as_float(lo), __uint_as_float(hi)), bias), a, b);
            out[i * 2 + h] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
        }
}
// four floats of shared memory, the same for all lanes
__device__ __forceinline__ void tl_load4(unsigned at, float* f) {
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]) : "r"(at));
}

}  // namespace

template <int D, bool Q8, bool PREFIX>
__global__ void __launch_bounds__((TlSizes<D, Q8>::THREADS), 1)
attention_tiles_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const float* __restrict__ ksc, const float* __restrict__ vsc,
                       const bf16* __restrict__ q, int q_stride, const int* __restrict__ block_table, int max_pages, int n_pages, const TlWork work, bf16* __restrict__ out,
                       int nh, int nkv, int page_size, float scale_log2e, int* __restrict__ err) {
    using Z = TlSizes<D, Q8>;
    constexpr int STAGES = Z::STAGES, TILE = Z::TILE, NA = D / 64;
    constexpr unsigned ATOM = TL_BN * 128, Q_ATOM = TL_BM * 128;
    // columns of tensor memory: outputs, scores, weights, and the queries of the first tile (of both where they fit)
    constexpr unsigned S_COL = 2 * D, P_COL = S_COL + 2 * TL_BN, Q_COL = P_COL + TL_BN, TMEM_COLS = 512;
    constexpr bool BOTH_Q = Q_COL + D <= TMEM_COLS;
    constexpr int SHARE_ROW = (D + 4) * 4;      // bytes of a row of a prefix's share: accumulators, maximum and sum
    static_assert(!PREFIX || 2 * TL_BM * (SHARE_ROW + TL_CLUSTER * 4) <= 2 * Z::Q_TILE + STAGES * 2 * TILE + Z::RAW * 2 * Z::RAW_TILE, "the shares must fit the tiles' memory");
    constexpr unsigned IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(TL_BN >> 3) << 17) | ((unsigned)(TL_BM >> 4) << 24);
    constexpr unsigned IDESC_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((unsigned)(D >> 3) << 17) | ((unsigned)(TL_BM >> 4) << 24);
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const unsigned base = tc_smem_u32(smem_raw);
    const unsigned q_s = base, kv_s = q_s + 2 * Z::Q_TILE, raw_s = kv_s + STAGES * 2 * TILE, sc_s = raw_s + Z::RAW * 2 * Z::RAW_TILE;
    const unsigned f_s = sc_s + Z::RAW * Z::SCALES;         // the factors of a block's scores and weights
    const unsigned bars0 = f_s + Z::RAW * Z::SCALES;
    const unsigned q_full = bars0, k_full0 = q_full + 8, k_empty0 = k_full0 + 8 * STAGES, v_full0 = k_empty0 + 8 * STAGES, v_empty0 = v_full0 + 8 * STAGES;
    const unsigned raw_full0 = v_empty0 + 8 * STAGES, raw_empty0 = raw_full0 + 8 * TL_RAW, s_full0 = raw_empty0 + 8 * TL_RAW, s_read0 = s_full0 + 16, p_full0 = s_read0 + 16, pv_done0 = p_full0 + 16, f_full0 = pv_done0 + 16;
    unsigned* holder = reinterpret_cast<unsigned*>(smem_raw + (f_full0 + 8 * TL_RAW - base));
    if ((base & 1023u) != 0) {          // cannot happen without static shared memory; never run misaligned
        if (threadIdx.x == 0) atomicExch(err, TC_ERR_MISALIGNED_SMEM);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, TL_SOFTMAX * 32);
        for (int i = 0; i < STAGES; i++) {
            mbar_init(k_full0 + 8 * i, Q8 ? 128 : 1);
            mbar_init(v_full0 + 8 * i, Q8 ? 128 : 1);
            mbar_init(k_empty0 + 8 * i, 2);        // both tiles
            mbar_init(v_empty0 + 8 * i, 2);
        }
        for (int i = 0; i < TL_RAW; i++) {
            mbar_init(raw_full0 + 8 * i, 1);
            mbar_init(raw_empty0 + 8 * i, 128);
            mbar_init(f_full0 + 8 * i, TL_BN);
        }
        for (int w = 0; w < 2; w++) {
            mbar_init(s_full0 + 8 * w, 1);
            mbar_init(s_read0 + 8 * w, TL_BM);
            mbar_init(p_full0 + 8 * w, TL_BM);
            mbar_init(pv_done0 + 8 * w, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == TL_MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(holder)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = *holder;
    if (PREFIX) {
        // in this order, for attention_pages.cu runs beside this kernel without a wait of its own: what comes before is through once it starts
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    } else {
        pdl_grid_sync();
    }

    // ---- which rows and keys
    const int G = nh / nkv;
    int member0 = 0;
    int hk, row0 = 0, n_rows, token0, past = 0, seq, jb0, last_key, nb[2], first_key;       // of the block: its rows, from row0 of its (sequence or tile)'s
    int4 tile = make_int4(0, 0, 0, 0);
    const int end = last_in_table(max_pages, page_size);
    if (PREFIX) {
        hk = blockIdx.y;
        member0 = blockIdx.z * (2 * TL_BM / G);
        const int first_member = work.members[member0];
        tile = work.tiles[blockIdx.z];
        if (tile.y - 1 > end) {
            if (threadIdx.x == 0) atomicExch(err, TL_ERR_PAGE);
            tile.y = end + 1;
        }
        n_rows = tile.x > 0 && tile.y > 0 ? min(tile.x, 2 * TL_BM / G) * G : 0;
        token0 = 0;
        seq = n_rows ? work.token_seq[first_member] : 0;
        const int all = (tile.y + TL_BN - 1) / TL_BN, per = (all + gridDim.x - 1) / gridDim.x;
        jb0 = blockIdx.x * per;
        first_key = jb0 * TL_BN;
        last_key = tile.y - 1;
        const int n = max(0, min(per, all - jb0));
        nb[0] = n_rows > 0 ? n : 0;
        nb[1] = n_rows > TL_BM ? n : 0;
    } else {
        // Blocks with the most keys before them start first: the longest sequences (of up to 128, by counting those that come before), and of each the last tile.
        // (Sixteen unequal prompts of 2,048 tokens together 70 us, in the order of the step 74.)
        hk = blockIdx.x;
        seq = blockIdx.z;
        if (gridDim.z > 1 && gridDim.z <= TL_ORDERED) {
            int* chosen = reinterpret_cast<int*>(holder + 1);
            const int n = gridDim.z, b = threadIdx.x;
            if (b < n) {
                const int len = work.seq_lens[b];
                int before = 0;
                for (int j = 0; j < n; j++) {
                    const int other = work.seq_lens[j];
                    before += other > len || (other == len && j < b);
                }
                if (before == (int)blockIdx.z) *chosen = b;
            }
            __syncthreads();
            seq = *chosen;
        }
        token0 = work.cu_q[seq];
        const int q_len = work.cu_q[seq + 1] - token0, all_rows = q_len * G;
        past = work.seq_lens[seq] - q_len;
        const int at = (all_rows + work.tile_rows - 1) / work.tile_rows - 1 - (int)blockIdx.y;
        row0 = at * work.tile_rows;
        n_rows = at < 0 ? 0 : min(work.tile_rows, all_rows - row0);
        first_key = n_rows > 0 ? max(0, first_visible(past + row0 / G, work.span)) : 0;
        jb0 = first_key / TL_BN;
        last_key = n_rows > 0 ? past + (row0 + n_rows - 1) / G : -1;
        nb[0] = n_rows > 0 ? min(past + (row0 + min(n_rows, TL_BM) - 1) / G, end) / TL_BN - jb0 + 1 : 0;
        nb[1] = n_rows > TL_BM ? min(last_key, end) / TL_BN - jb0 + 1 : 0;
        if (last_key > end && threadIdx.x == 0) atomicExch(err, TL_ERR_PAGE);
    }
    const int n_blocks = max(nb[0], nb[1]);         // the second tile, where it has rows, sees at least as far as the first

    if (warp == TL_TMA_WARP) {
        // ---- pages.  One that the sequence does not hold is reported and another read in its place.
        if (lane == 0) {
            const int* bt = block_table + (size_t)seq * max_pages;
            for (int i = 0; i < n_blocks; i++) {
                const int key0 = (jb0 + i) * TL_BN;
                int page = key0 / page_size < max_pages ? bt[key0 / page_size] : -1;
                if (page < 0 || page >= n_pages) {
                    atomicExch(err, TL_ERR_PAGE);
                    page = 0;
                }
                const int row = (page * nkv + hk) * page_size + key0 % page_size;
                if (Q8) {
                    const int st = i % TL_RAW;
                    if (i >= TL_RAW && !mbar_wait(raw_empty0 + 8 * st, ((i / TL_RAW) - 1) & 1, err, TC_ERR_TIMEOUT_PREFILL)) break;
                    const unsigned bar = raw_full0 + 8 * st, dst = raw_s + st * 2 * Z::RAW_TILE;
                    mbar_expect_tx(bar, 2 * Z::RAW_TILE + Z::SCALES);
                    tma_load_2d(dst, &map_k, 0, row, bar);
                    rows_bulk(sc_s + st * Z::SCALES, ksc + row, TL_BN * 4, bar);
                    tma_load_2d(dst + Z::RAW_TILE, &map_v, 0, row, bar);
                    rows_bulk(sc_s + st * Z::SCALES + TL_BN * 4, vsc + row, TL_BN * 4, bar);
                } else {
                    const int st = i % STAGES;
                    const unsigned kd = kv_s + st * 2 * TILE, vd = kd + TILE;
                    if (i >= STAGES && !mbar_wait(k_empty0 + 8 * st, ((i / STAGES) - 1) & 1, err, TC_ERR_TIMEOUT_PREFILL)) break;
                    mbar_expect_tx(k_full0 + 8 * st, TILE);
                    for (int a = 0; a < NA; a++) tma_load_2d(kd + a * ATOM, &map_k, 64 * a, row, k_full0 + 8 * st);
                    if (i >= STAGES && !mbar_wait(v_empty0 + 8 * st, ((i / STAGES) - 1) & 1, err, TC_ERR_TIMEOUT_PREFILL)) break;
                    mbar_expect_tx(v_full0 + 8 * st, TILE);
                    for (int a = 0; a < NA; a++) tma_load_2d(vd + a * ATOM, &map_v, 64 * a, row, v_full0 + 8 * st);
                }
            }
        }
    } else if (warp == TL_MMA_WARP || warp == TL_MMA_WARP + 1) {
        // ---- products, a warp for each tile (one for both was busy with its waits and commits for longer than a softmax).  The scores of block i + 1 are made
        // as soon as the softmax has taken those of block i into its registers, and so are there when it comes back.  The warp stays together around what one
        // lane issues, so that descriptors lie in uniform registers (a lane by itself took 95 clocks for each instruction).
        const int w = warp - TL_MMA_WARP, nbw = nb[w];
        const bool elected = elect_one(), q_in_tmem = w == 0 || BOTH_Q;
        const unsigned long long q_desc = desc_kmajor(q_s + w * Z::Q_TILE), k_desc = desc_kmajor(kv_s), v_desc = desc_mnmajor(kv_s + TILE, ATOM);
        const unsigned s_at = tmem + S_COL + w * TL_BN, p_at = tmem + P_COL + w * (TL_BN / 2), o_at = tmem + w * D, q_at = tmem + Q_COL + w * (D / 2);
        auto wait = [&](unsigned bar, int phase) { return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, err, TC_ERR_TIMEOUT_PREFILL)) != 0; };
        auto scores = [&](int i) {
            const int st = i % STAGES;
            if (!wait(k_full0 + 8 * st, i / STAGES)) return false;
            if (i >= nbw) {                                  // the other tile's alone
                if (elected) tl_arrive(k_empty0 + 8 * st);
                return true;
            }
            if (i > 0 && !wait(s_read0 + 8 * w, i - 1)) return false;
            tc_fence_after();
            if (elected) {
                const unsigned long long kd = k_desc + (unsigned)st * (2 * TILE >> 4);
                if (q_in_tmem) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; kk++) mma_bf16_ts(s_at, q_at + kk * 8, kd + (kk >> 2) * (ATOM >> 4) + (kk & 3) * 2, IDESC_S, kk > 0);
                } else {
#pragma unroll
                    for (int kk = 0; kk < D / 16; kk++)
                        mma_bf16_ss(s_at, q_desc + (kk >> 2) * (Q_ATOM >> 4) + (kk & 3) * 2, kd + (kk >> 2) * (ATOM >> 4) + (kk & 3) * 2, IDESC_S, kk > 0);
                }
                mma_commit(s_full0 + 8 * w);
                mma_commit(k_empty0 + 8 * st);
            }
            return true;
        };
        bool alive = n_blocks > 0 && wait(q_full, 0) && scores(0);
        for (int i = 0; i < n_blocks && alive; i++) {
            if (i + 1 < n_blocks && !(alive = scores(i + 1))) break;
            const int st = i % STAGES;
            if (!(alive = wait(v_full0 + 8 * st, i / STAGES))) break;
            if (i >= nbw) {
                if (elected) tl_arrive(v_empty0 + 8 * st);
                continue;
            }
            if (!(alive = wait(p_full0 + 8 * w, i))) break;
            tc_fence_after();
            if (elected) {
                const unsigned long long vd = v_desc + (unsigned)st * (2 * TILE >> 4);
#pragma unroll
                for (int ks = 0; ks < TL_BN / 16; ks++) mma_bf16_ts(o_at, p_at + ks * 8, vd + ks * (16 * 128 >> 4), IDESC_O, (i > 0 || ks > 0) ? 1u : 0u);
                mma_commit(pv_done0 + 8 * w);
                mma_commit(v_empty0 + 8 * st);
            }
        }
    } else if (Q8 && warp >= TL_WIDEN_WARP) {
        // ---- bytes to bfloat16, and the factors of the scores (with the softmax's scale) and of the weights.  Keys outside the block's range, where
        // another sequence's may lie, have factors of zero.  The ring of factors has four places: those of block i + 4 are made behind
        // the wait for the stage of V(i + 2), which the products of block i leave (v_empty of both tiles), so behind every softmax of block i.
        const int ct = threadIdx.x - TL_WIDEN_WARP * 32;
        auto widen = [&](const unsigned char* raw, unsigned dst) {
#pragma unroll
            for (int it = 0; it < TL_BN * D / 16 / 128; it++) {
                const int id = ct + it * 128, rest = id >> 3;
                const int r = (D == 128 ? rest >> 1 : rest) * 2 ^ ((id & 4) ? 5 : 0), c = (id & 3) + (D == 128 ? (rest & 1) * 4 : 0);
                const uint4 v = *reinterpret_cast<const uint4*>(raw + (D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + c * 16));
                const unsigned w[4] = {v.x, v.y, v.z, v.w};
                unsigned o[8];
                tl_widen(w, o);
                const unsigned at = dst + (c >> 2) * ATOM + r * 128, p = (c & 3) * 2;
                tl_store16(at + ((p ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
                tl_store16(at + (((p + 1) ^ (r & 7)) << 4), o[4], o[5], o[6], o[7]);
            }
        };
        // in the order in which the products ask for them: K(0), K(1), V(0), K(2), V(1), ...
        auto keys = [&](int i) {
            const int rs = i % TL_RAW, st = i % STAGES, key0 = (jb0 + i) * TL_BN;
            if (!mbar_wait(raw_full0 + 8 * rs, (i / TL_RAW) & 1, err, TC_ERR_TIMEOUT_PREFILL)) return false;
            if (ct < TL_BN) {
                const float* ks = reinterpret_cast<const float*>(smem_raw + (sc_s - base) + rs * Z::SCALES);
                const float* vs = ks + TL_BN;
                const bool in = key0 + ct >= first_key && key0 + ct <= last_key, number = fabsf(ks[ct]) < INFINITY && fabsf(vs[ct]) < INFINITY;
                float* f = reinterpret_cast<float*>(smem_raw + (f_s - base) + rs * Z::SCALES);
                f[ct] = !in ? 0.f : number ? ks[ct] * scale_log2e : __uint_as_float(0x7fffffffu);
                f[TL_BN + ct] = in && number ? vs[ct] : 0.f;
                tl_arrive(f_full0 + 8 * rs);
            }
            if (i >= STAGES && !mbar_wait(k_empty0 + 8 * st, ((i / STAGES) - 1) & 1, err, TC_ERR_TIMEOUT_PREFILL)) return false;
            widen(smem_raw + (raw_s - base) + rs * 2 * Z::RAW_TILE, kv_s + st * 2 * TILE);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tl_arrive(k_full0 + 8 * st);
            return true;
        };
        bool alive = n_blocks > 0 && keys(0);
        for (int i = 0; i < n_blocks && alive; i++) {
            if (i + 1 < n_blocks && !(alive = keys(i + 1))) break;
            const int rs = i % TL_RAW, st = i % STAGES;
            if (i >= STAGES && !(alive = mbar_wait(v_empty0 + 8 * st, ((i / STAGES) - 1) & 1, err, TC_ERR_TIMEOUT_PREFILL))) break;
            widen(smem_raw + (raw_s - base) + rs * 2 * Z::RAW_TILE + Z::RAW_TILE, kv_s + st * 2 * TILE + TILE);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tl_arrive(v_full0 + 8 * st);
            tl_arrive(raw_empty0 + 8 * rs);
        }
    } else if (warp < TL_SOFTMAX) {
        // ---- softmax: thread = row = lane of tensor memory
        const int w = warp >> 2, r = threadIdx.x & 127, br = w * TL_BM + r;       // br: row of the block
        const bool valid = br < n_rows;
        int token = 0, h = hk * G, pos = last_key;
        if (valid) {
            if (PREFIX) {
                token = work.members[member0 + br / G];
                h = hk * G + br % G;
            } else {
                const int i = (row0 + br) / G;
                token = token0 + i;
                h = hk * G + (row0 + br) % G;
                pos = past + i;
            }
        }
        const unsigned lane_addr = tmem + ((unsigned)((warp & 3) * 32) << 16), s_addr = lane_addr + S_COL + w * TL_BN, p_addr = lane_addr + P_COL + w * (TL_BN / 2),
                       o_addr = lane_addr + w * D;
        // the queries into a swizzled tile of shared memory, whole rows at a time, and the first tile's from there into tensor memory; rows behind the last one are
        // zeros
        {
            const long long mine = valid ? (long long)token * q_stride + (long long)h * D : -1;
            const unsigned tile_s = q_s + w * Z::Q_TILE;
            constexpr int LINE = D / 8, ROWS = 32 / LINE;           // lanes of a row, rows at a time
            // (asynchronous copies, in a loop that stays one: unrolled, its instructions alone, fetched anew by every block's first warps, took longer than the rows)
            const int c = lane % LINE;
#pragma unroll 1
            for (int k = 0; k < LINE; k++) {
                const int rr = k * ROWS + lane / LINE, row = (warp & 3) * 32 + rr;
                const long long from = __shfl_sync(0xffffffffu, mine, rr);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tile_s + (c >> 3) * Q_ATOM + row * 128 + (((c & 7) ^ (row & 7)) << 4)),
                             "l"(q + (from >= 0 ? from : 0) + c * 8), "r"(from >= 0 ? 16 : 0) : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (w == 0 || BOTH_Q) {
                __syncwarp();
#pragma unroll 1
                for (int c0 = 0; c0 < D / 64; c0++) {
                    unsigned x[32];
#pragma unroll
                    for (int c = 0; c < 8; c++)
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[c * 4]), "=r"(x[c * 4 + 1]), "=r"(x[c * 4 + 2]), "=r"(x[c * 4 + 3])
                                     : "r"(tile_s + c0 * Q_ATOM + r * 128 + ((c ^ (r & 7)) << 4)) : "memory");
                    tmem_st32(lane_addr + Q_COL + w * (D / 2) + c0 * 32, x);
                }
                tmem_wait_st();
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc_fence_before();
            tl_arrive(q_full);
        }
        const int nbw = nb[w];
        // what the tile's rows see: everything in blocks between the last row's first key and the first row's last one
        const int tile_first = PREFIX ? last_key : past + (row0 + w * TL_BM) / G, tile_last = PREFIX ? last_key : past + (row0 + min(n_rows, (w + 1) * TL_BM) - 1) / G;
        const int lo_pos = PREFIX ? 0 : nbw > 0 ? first_visible(pos, work.span) : 0, lo_last = PREFIX || nbw == 0 ? 0 : first_visible(tile_last, work.span);
        const float unit = Q8 ? 1.f : scale_log2e;
        float m_ref = -INFINITY, l_run = 0.f;
        bool alive = true;
        for (int i = 0; i < nbw; i++) {
            const int key0 = (jb0 + i) * TL_BN;
            alive = __all_sync(0xffffffffu, mbar_wait(s_full0 + 8 * w, i & 1, err, TC_ERR_TIMEOUT_PREFILL));
            if (!alive) break;
            tc_fence_after();
            unsigned sr[TL_BN];
            tmem_ld32_issue(s_addr, sr);
            tmem_ld32_issue(s_addr + 32, sr + 32);
            tmem_wait_ld<TL_BN>(sr);
            tc_fence_before();
            tl_arrive(s_read0 + 8 * w);
            const unsigned f_at = f_s + (i % TL_RAW) * Z::SCALES;
            if (Q8) {
                alive = __all_sync(0xffffffffu, mbar_wait(f_full0 + 8 * (i % TL_RAW), (i / TL_RAW) & 1, err, TC_ERR_TIMEOUT_PREFILL));
                if (!alive) break;
#pragma unroll
                for (int c = 0; c < TL_BN; c += 4) {
                    float f[4], x[4];
                    tl_load4(f_at + c * 4, f);
                    f2_unpack(f2_mul(f2_pack(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), f2_pack(f[0], f[1])), x[0], x[1]);
                    f2_unpack(f2_mul(f2_pack(__uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3])), f2_pack(f[2], f[3])), x[2], x[3]);
#pragma unroll
                    for (int e = 0; e < 4; e++) sr[c + e] = __float_as_uint(x[e]);
                }
            }
            if (key0 + TL_BN - 1 > tile_first || key0 < lo_last) {
#pragma unroll
                for (int c = 0; c < TL_BN; c++)
                    if (key0 + c > pos || key0 + c < lo_pos) sr[c] = 0xff800000u;      // -inf
            }
            float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
            for (int c = 0; c < TL_BN; c += 8) {
                mx0 = max3(mx0, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
                mx1 = max3(mx1, __uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3]));
                mx2 = max3(mx2, __uint_as_float(sr[c + 4]), __uint_as_float(sr[c + 5]));
                mx3 = max3(mx3, __uint_as_float(sr[c + 6]), __uint_as_float(sr[c + 7]));
            }
            const float m_new = fmaxf(m_ref, fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * unit);
            const bool grown = m_new > m_ref + TL_RESCALE_STEP;      // true for m_ref = -inf, m_new finite
            // the products of the block before: their weights lie where this block's go, and the output may be touched
            if (i > 0 && !(alive = __all_sync(0xffffffffu, mbar_wait(pv_done0 + 8 * w, (i - 1) & 1, err, TC_ERR_TIMEOUT_PREFILL)))) break;
            if (__any_sync(0xffffffffu, grown)) {
                if (i > 0) {
                    const float corr = m_new == -INFINITY ? 1.f : m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - m_new);
                    tc_fence_after();
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        unsigned o[32];
                        tmem_ld32_issue(o_addr + c0, o);
                        tmem_wait_ld<32>(o);
#pragma unroll
                        for (int c = 0; c < 32; c++) o[c] = __float_as_uint(__uint_as_float(o[c]) * corr);
                        tmem_st32(o_addr + c0, o);
                    }
                    tmem_wait_st();
                    l_run *= corr;
                }
                m_ref = m_new;
            }
            const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
            unsigned pr[TL_BN / 2];
            const unsigned long long scale2 = f2_pack(unit, unit), neg_m2 = f2_pack(-m_use, -m_use);
            unsigned long long psa = f2_pack(0.f, 0.f), psb = psa;
#pragma unroll
            for (int c = 0; c < TL_BN; c += 4) {
                float x0, x1, x2, x3;
                f2_unpack(f2_fma(f2_pack(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), scale2, neg_m2), x0, x1);
                f2_unpack(f2_fma(f2_pack(__uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3])), scale2, neg_m2), x2, x3);
                const float p0 = fast_exp2(x0), p1 = fast_exp2(x1), p2 = fast_exp2(x2), p3 = fast_exp2(x3);
                psa = f2_add(psa, f2_pack(p0, p1));
                psb = f2_add(psb, f2_pack(p2, p3));
                if (Q8) {
                    float f[4], w0, w1, w2, w3;
                    tl_load4(f_at + TL_BN * 4 + c * 4, f);
                    f2_unpack(f2_mul(f2_pack(p0, p1), f2_pack(f[0], f[1])), w0, w1);
                    f2_unpack(f2_mul(f2_pack(p2, p3), f2_pack(f[2], f[3])), w2, w3);
                    pr[c >> 1] = pack_bf16(w0, w1);
                    pr[(c >> 1) + 1] = pack_bf16(w2, w3);
                } else {
                    pr[c >> 1] = pack_bf16(p0, p1);
                    pr[(c >> 1) + 1] = pack_bf16(p2, p3);
                }
            }
            {
                float a0, a1, b0, b1;
                f2_unpack(psa, a0, a1);
                f2_unpack(psb, b0, b1);
                l_run += (a0 + a1) + (b0 + b1);
            }
            tmem_st32(p_addr, pr);
            tmem_wait_st();
            if (!Q8 && key0 + TL_BN - 1 > last_key) {
                // behind the prefix the page may hold anything: those rows of V are cleared (both tiles write the same zeros)
                const int st = i % STAGES;
                alive = __all_sync(0xffffffffu, mbar_wait(v_full0 + 8 * st, (i / STAGES) & 1, err, TC_ERR_TIMEOUT_PREFILL));
                if (r < TL_BN && key0 + r > last_key)
#pragma unroll
                    for (int a = 0; a < NA; a++)
#pragma unroll
                        for (int c = 0; c < 8; c++) tl_store16(kv_s + st * 2 * TILE + TILE + a * ATOM + r * 128 + c * 16, 0u, 0u, 0u, 0u);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            if (!alive) break;
            tc_fence_before();
            tl_arrive(p_full0 + 8 * w);
        }
        if (alive && nbw > 0) alive = __all_sync(0xffffffffu, mbar_wait(pv_done0 + 8 * w, (nbw - 1) & 1, err, TC_ERR_TIMEOUT_PREFILL));
        const size_t head = (size_t)token * nh + h;
        if (PREFIX) {
            // the block's share of a row into shared memory: all products of both tiles have to be through with what lies there
            asm volatile("bar.sync 1, %0;" ::"n"(TL_SOFTMAX * 32) : "memory");
            const unsigned dst = base + br * SHARE_ROW;
            if (nbw > 0) {
                tc_fence_after();
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    unsigned o[32];
                    tmem_ld32_issue(o_addr + c0, o);
                    tmem_wait_ld<32>(o);
#pragma unroll
                    for (int c = 0; c < 32; c += 4) tl_store16(dst + (c0 + c) * 4, o[c], o[c + 1], o[c + 2], o[c + 3]);
                }
            }
            tl_store16(dst + D * 4, __float_as_uint(nbw > 0 ? m_ref : -INFINITY), __float_as_uint(nbw > 0 ? l_run : 0.f), 0u, 0u);
        } else if (alive) {
            // (a row that sees nothing, one before the first position of its sequence, is zeros)
            tc_fence_after();
            const float inv = nbw > 0 && l_run != 0.f ? 1.0f / l_run : 0.f;
            bf16* dst = out + head * D;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                unsigned o[32] = {};
                if (nbw > 0) {
                    tmem_ld32_issue(o_addr + c0, o);
                    tmem_wait_ld<32>(o);
                }
                if (valid)
#pragma unroll
                    for (int c = 0; c < 32; c += 8) {
                        float f[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) f[e] = __uint_as_float(o[c + e]) * inv;
                        store8(dst + c0 + c, f);
                    }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PREFIX) {
        // the cluster's shares of a row (ascending) become one; every block makes a part of the rows: first their factors, then four columns to a thread
        const int n = work.cluster, rank = (int)blockIdx.x % n, rows_each = (n_rows + n - 1) / n, r0 = rank * rows_each, r1 = min(n_rows, r0 + rows_each);
        const unsigned factors = base + 2 * TL_BM * SHARE_ROW;              // [row of the part][TL_CLUSTER]
        if (n > 1) rows_cluster_sync();
        for (int br = r0 + (int)threadIdx.x; br < r1; br += (int)blockDim.x) {
            float4 ml[TL_CLUSTER];
            float M = -INFINITY, f[TL_CLUSTER], den = 0.f;
#pragma unroll
            for (int k = 0; k < TL_CLUSTER; k++) {
                ml[k] = k < n ? rows_remote4(base + br * SHARE_ROW + D * 4, k) : make_float4(-INFINITY, 0.f, 0.f, 0.f);
                M = fmaxf(M, ml[k].x);
            }
#pragma unroll
            for (int k = 0; k < TL_CLUSTER; k++) {
                // (no keys: no factor; a sum that is no number goes on)
                f[k] = ml[k].y == 0.f ? 0.f : ml[k].x == -INFINITY ? 1.f : fast_exp2(ml[k].x - M);
                if (ml[k].y != 0.f) den += f[k] * ml[k].y;
            }
            tl_store16(factors + (br - r0) * (TL_CLUSTER * 4), __float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
            const size_t share = ((size_t)work.members[member0 + br / G] * nh + hk * G + br % G) * work.slots + work.slot0 + blockIdx.x / n;
            *reinterpret_cast<float2*>(work.part_ml + share * 2) = make_float2(M, den);
        }
        __syncthreads();
#pragma unroll 2
        for (int idx = (int)threadIdx.x; idx < (r1 - r0) * (D / 4); idx += (int)blockDim.x) {
            const int i = idx / (D / 4), br = r0 + i, c = idx % (D / 4);
            float f[TL_CLUSTER];
            tl_load4(factors + i * (TL_CLUSTER * 4), f);
            float4 v[TL_CLUSTER], num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < TL_CLUSTER; k++)
                if (f[k] != 0.f) v[k] = rows_remote4(base + br * SHARE_ROW + c * 16, k);
#pragma unroll
            for (int k = 0; k < TL_CLUSTER; k++) {
                if (f[k] == 0.f) continue;
                num.x += f[k] * v[k].x;
                num.y += f[k] * v[k].y;
                num.z += f[k] * v[k].z;
                num.w += f[k] * v[k].w;
            }
            const size_t share = ((size_t)work.members[member0 + br / G] * nh + hk * G + br % G) * work.slots + work.slot0 + blockIdx.x / n;
            *reinterpret_cast<float4*>(work.part_acc + share * D + c * 4) = num;
        }
        if (n > 1) rows_cluster_sync();               // the others may still read this block's rows
    }
    if (warp == TL_MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// ---- host side

template <int D, bool Q8, bool PREFIX>
static int tl_launch(dim3 grid, const void* q, int q_stride, const void* kc, const void* vc, const float* ksc, const float* vsc, long long n_pages, const int* block_table,
                     int max_pages, const TlWork& work, void* out, int nh, int nkv, int page_size, float scale, int* err, cudaStream_t s) {
    CUtensorMap mk, mv;
    const long long rows = n_pages * nkv * page_size;
    const CUtensorMapSwizzle swizzle = Q8 && D == 64 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B;
    int rc;
    if ((rc = rows_make_map(&mk, kc, rows, D, TL_BN, Q8, swizzle)) || (rc = rows_make_map(&mv, vc, rows, D, TL_BN, Q8, swizzle))) return rc;
    auto kern = attention_tiles_kernel<D, Q8, PREFIX>;
    const int smem = TlSizes<D, Q8>::SMEM;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    return illm_launch_cluster(kern, grid, dim3(TlSizes<D, Q8>::THREADS), PREFIX ? work.cluster : 1, smem, s, mk, mv, ksc, vsc, (const bf16*)q, q_stride, block_table, max_pages,
                               (int)n_pages, work, (bf16*)out, nh, nkv, page_size, scale * 1.4426950408889634f, err);
}

static bool tl_bad(const void* q, int q_stride, const void* kc, const void* vc, const float* ksc, const float* vsc, long long n_pages, int max_pages, int nh, int nkv, int page_size,
                   const int* err) {
    return nkv <= 0 || nh <= 0 || nh % nkv || nkv > 65535 || (q_stride & 7) || page_size <= 0 || page_size % TL_BN || max_pages <= 0 || n_pages <= 0 ||
           n_pages * nkv * page_size > 0x7fffffffLL || !q || ((uintptr_t)q & 15) || !kc || !vc || ((uintptr_t)kc & 15) || ((uintptr_t)vc & 15) || (!ksc) != (!vsc) ||
           ((uintptr_t)ksc & 15) || ((uintptr_t)vsc & 15) || !err;
}

// Prompts over rows of eight bits: q, rows of q_stride bfloat16 elements whose first nh * d are the query heads; kc, vc one entry's pages of bytes
// [n_pages, nkv, page_size, d] and their scales; cu_q [B + 1], seq_lens [B] as for attention_prefill_tc; out [T, nh * d].  tile_rows: 128, 256 or 0 (by a rule).
// d 64 or 128, page_size a multiple of 64.  span: see first_visible.  err: 5 a wait ran out, 6 shared memory, 8 a visible position without a page.
extern "C" int illm_attention_tiles_int8(const void* q, int q_stride, const void* kc, const void* vc, const float* ksc, const float* vsc, long long n_pages,
                                         const int* block_table, int max_pages, const int* cu_q, const int* seq_lens, void* out, int B, int max_q, int nh, int nkv, int d,
                                         int page_size, int span, float scale, int tile_rows, int* err, void* stream) {
    if (B <= 0 || max_q <= 0) return 0;
    if (tl_bad(q, q_stride, kc, vc, ksc, vsc, n_pages, max_pages, nh, nkv, page_size, err) || !ksc || B > 65535 || (tile_rows && tile_rows != TL_BM && tile_rows != 2 * TL_BM) || !out ||
        ((uintptr_t)out & 15))
        return ILLM_ERR_BAD_ARG;
    // two tiles a block over the same keys, or one while that leaves SMs without a block (32 / 8 heads: one prompt of 200 tokens 8.7 us with one tile, 11.3 with two;
    // sixteen of 2,048 together 93 and 70)
    if (tile_rows == 0) tile_rows = ((long long)max_q * (nh / nkv) + 2 * TL_BM - 1) / (2 * TL_BM) * nkv * B < illm_sm_count() ? TL_BM : 2 * TL_BM;
    const long long tiles = ((long long)max_q * (nh / nkv) + tile_rows - 1) / tile_rows;
    if (tiles > 65535 || (long long)max_q * (nh / nkv) > 0x7fffffffLL) return ILLM_ERR_BAD_ARG;
    TlWork work = {};
    work.cu_q = cu_q;
    work.seq_lens = seq_lens;
    work.span = span;
    work.tile_rows = tile_rows;
    const dim3 grid((unsigned)nkv, (unsigned)tiles, (unsigned)B);
    cudaStream_t s = (cudaStream_t)stream;
    if (d == 128) return tl_launch<128, true, false>(grid, q, q_stride, kc, vc, ksc, vsc, n_pages, block_table, max_pages, work, out, nh, nkv, page_size, scale, err, s);
    if (d == 64) return tl_launch<64, true, false>(grid, q, q_stride, kc, vc, ksc, vsc, n_pages, block_table, max_pages, work, out, nh, nkv, page_size, scale, err, s);
    return ILLM_ERR_BAD_ARG;
}

// Parts of a prefix that are joined before they leave: up to four, whole clusters.
extern "C" int illm_attention_tiles_cluster(int splits) { return splits < TL_CLUSTER ? (splits < 1 ? 1 : splits) : splits % TL_CLUSTER == 0 ? TL_CLUSTER : splits % 2 == 0 ? 2 : 1; }

// The shares of common prefixes (ksc, vsc nullptr: bfloat16 pages): for every tile of the plan (at most 256 / (nh / nkv) members), whose positions are cut into `splits` parts,
// of which every c = illm_attention_tiles_cluster(splits) are joined: for every (member, head) accumulators, maximum (in units of log2) and sum at share slot0 + part / c of
// `slots`: part_acc float [T, nh, slots, d], part_ml float [T, nh, slots, 2].  illm_attention_pages adds them up with a token's own.  bfloat16 rows: a scale below zero
// is refused (the softmax takes its reference from the largest score before the scale).
extern "C" int illm_attention_tiles_prefix(const void* q, int q_stride, const void* kc, const void* vc, const float* ksc, const float* vsc, long long n_pages,
                                           const int* block_table, int max_pages, const int* token_seq, const int* plan_tiles, const int* plan_members, int n_tiles,
                                           float* part_acc, float* part_ml, int nh, int nkv, int d, int page_size, float scale, int slots, int slot0, int splits, int* err,
                                           void* stream) {
    if (n_tiles <= 0) return 0;
    if (tl_bad(q, q_stride, kc, vc, ksc, vsc, n_pages, max_pages, nh, nkv, page_size, err) || nh / nkv > 2 * TL_BM || n_tiles > 65535 || splits < 1 || splits > 256 ||
        (!ksc && !(scale >= 0.f)) || slot0 < 0 || slot0 + splits / illm_attention_tiles_cluster(splits) > slots || !part_acc || !part_ml || ((uintptr_t)part_acc & 15) || ((uintptr_t)part_ml & 7) || !plan_tiles || ((uintptr_t)plan_tiles & 15) || !plan_members)
        return ILLM_ERR_BAD_ARG;
    TlWork work = {};
    work.tiles = reinterpret_cast<const int4*>(plan_tiles);
    work.members = plan_members;
    work.token_seq = token_seq;
    work.slots = slots;
    work.slot0 = slot0;
    work.cluster = illm_attention_tiles_cluster(splits);
    work.part_acc = part_acc;
    work.part_ml = part_ml;
    const dim3 grid((unsigned)splits, (unsigned)nkv, (unsigned)n_tiles);
    cudaStream_t s = (cudaStream_t)stream;
#define TL_CASE(DD, QQ)                                                                                                                                           \
    if (d == DD && (ksc != nullptr) == QQ)                                                                                                                        \
        return tl_launch<DD, QQ, true>(grid, q, q_stride, kc, vc, ksc, vsc, n_pages, block_table, max_pages, work, nullptr, nh, nkv, page_size, scale, err, s);
    TL_CASE(128, true) TL_CASE(64, true) TL_CASE(128, false) TL_CASE(64, false)
#undef TL_CASE
    return ILLM_ERR_BAD_ARG;
}
