// Attention of single tokens over paged caches on warp-level tensor instructions, the keys as a stream: over rows of eight bits
// (kv_int8.cu) or bfloat16, and over positions that several sequences hold in common, which are read once for all of them.
//
//   o = sum_j p_j v_j,  p = softmax over the visible j of scale q . k_j       (src/kern/naive/naive.cpp:576-604, :531-553, :209-240, :634-662)
//
// The rows of a block's products are queries that walk the same keys: the heads of one token that share a key/value head or, for
// a common prefix, those of up to 16 / group of its tokens.  A block takes every n-th tile of 64 keys of its range.  One thread
// brings them by TMA into a ring of stages (swizzled; pages are multiples of 64 positions, so a tile lies in one page), four warps
// take 16 keys of a tile each, with a running maximum and sum of their own, and are joined at the end; the shares of all blocks of a
// head are joined by a second kernel in ascending order.  With a plan (common prefixes) the first blocks of the grid walk the
// prefixes and the others what every token has for itself behind its prefix, in one launch.
//
// Eight-bit rows.  A key's products are made from the bytes: 0x64 in front of a byte is 1024 + u in half precision, minus 1152 is
// u - 128 exactly, so a pair of elements costs a byte permutation and a subtraction, and for the values the permutation also makes
// the transposition that the product wants.  The queries are scaled by a power of two per row so that bfloat16 turns into
// half precision without loss (elements below 2^-24 of the row's largest lose bits), the key's scale is a factor of its score.  The
// values' scale goes into the softmax weight: w_j = 2^(s_j + log2 s^v_j - m'), with a maximum m' of its own next to the softmax's m,
// so that the largest weight of a row is 1 whatever the scales are; weights are rounded to half precision (2^-12 of a weight; those below 2^-24 of
// the largest to 2^-25 of it).  The sum of 2^(s_j - m), scores and accumulators are float32.
// A tile's hidden keys have weight 0 whatever lies there: bytes are finite, scales of hidden keys are not used.
// Bound by the rows' way from memory where sequences are long: 64 of up to 8,192 positions of 8 kv heads of 128 take 118 us, 0.87 of the copy rate; 8 of up to 4,096 of 32
// 39.7 us, 0.71.
// bfloat16 rows go as in attention_decode_ring.cu, which is the faster one without a plan (it also rotates and writes).
#include <cuda.h>
#include <cuda_fp16.h>
#include <math.h>

#include "paged_rows.cuh"
#include "tc_common.cuh"

#define PG_BN 64                        // keys per tile
#define PG_CONSUMERS 4
#define PG_THREADS ((PG_CONSUMERS + 1) * 32)
#define PG_MAX_SPLITS 32
#define PG_MAX_CLUSTER 8               // blocks whose shares are joined through shared memory
#define PG_ERR_PAGE 8                   // a visible position without a page
#define PG_AHEAD 8.0f                   // how far (in powers of two) a score may run ahead of what its weights are relative to

namespace {

__device__ __forceinline__ void pg_ldm(unsigned* r, unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void pg_ldm_t(unsigned* r, unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <bool HALF> __device__ __forceinline__ void pg_mma(float* c, const unsigned* a, unsigned b0, unsigned b1) {
    if (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pg_half2(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ unsigned pg_bf162(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
}
// two bytes of w (the selector names them; 4 is the 0x64 above them) as u - 128 in half precision
__device__ __forceinline__ unsigned pg_widen(unsigned w, unsigned selector) {
    unsigned r = __byte_perm(w, 0x64646464u, selector);
    const unsigned bias = 0x64806480u;       // 1152, twice
    __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&r), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const unsigned*>(&v);
}
// an 8 x 8 matrix of 16-bit elements, transposed
__device__ __forceinline__ unsigned pg_transpose(unsigned x) {
    unsigned y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float pg_log2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Byte offset of the 16-byte piece c of key row r inside a tile.  bfloat16: boxes of 64 channels of 8 KB, rows of 128 bytes, the
// piece's number XORed with the row's; eight bits: rows of D bytes, the same swizzle for 128 and the 64-byte one for 64.
template <int D, bool Q8> __device__ __forceinline__ unsigned pg_off(int r, int c) {
    if (!Q8) return (unsigned)((c >> 3) * (PG_BN * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
    if (D == 128) return (unsigned)(r * 128 + ((c ^ (r & 7)) << 4));
    return (unsigned)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}
// two floats of the same place in another block of the cluster
__device__ __forceinline__ float2 pg_remote2(unsigned at, unsigned rank) {
    unsigned a;
    float2 f;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(f.x), "=f"(f.y) : "r"(a) : "memory");
    return f;
}
__device__ __forceinline__ void pg_add(float4& sum, float4 v, float f) {
    sum.x += v.x * f;
    sum.y += v.y * f;
    sum.z += v.z * f;
    sum.w += v.w * f;
}
// four channels of a result; a row without keys is zeros
__device__ __forceinline__ void pg_result(bf16* to, float4 num, float den) {
    const bool none = den == 0.f;
    *reinterpret_cast<uint2*>(to) = make_uint2(pg_bf162(none ? 0.f : num.x / den, none ? 0.f : num.y / den), pg_bf162(none ? 0.f : num.z / den, none ? 0.f : num.w / den));
}

}  // namespace

// A plan of common prefixes (attention_decode_shared): int32 on the device.  `start` [T]: the positions that a token leaves to its
// group; `tiles` [n_tiles][4]: number of members, positions of the prefix, 0, 0; `members` [n_tiles][per_tile]: tokens.
struct PgPlan {
    const int* start;
    const int4* tiles;
    const int* members;
    int n_tiles, per_tile;
};

// Stages: as many as leave four blocks to an SM (five at head size 64, three of bfloat16 rows), or with sixteen rows, whose registers leave two blocks, more.  The blocks
// are short (one takes a few tiles after it has waited for its first), so that more of them are worth more than deeper rings: 64 sequences of 32 kv heads at
// 300 keys 46.7 us with two blocks of six stages, 38.3 with three of four, 37.1 with four of three (64 sequences of 8 kv heads at up to 8,192 keys 130, 115 and 118).
template <int D, bool Q8, int NT> struct PgRing {
    static constexpr int TILE = PG_BN * D * (Q8 ? 1 : 2), SCALES = Q8 ? 2 * PG_BN * 4 : 0;
    static constexpr int STAGES = !Q8 ? 256 / D : NT == 1 ? (D == 128 ? 3 : 4) : (D == 128 ? 4 : 6), BYTES = STAGES * (2 * TILE + SCALES) + 1024;
};

// grid: prefix tiles times kv heads times pre_splits, then tokens times kv heads times own_splits.  Shares: part_acc [T, nh, slots, D], part_ml [T, nh, slots, 2] with slots = own_splits + pre_splits,
// a token's own first.  No part_acc: the blocks of a (token, kv head) are a cluster that joins them through shared memory and writes `out`.
template <int D, bool Q8, int NT>
__global__ void __launch_bounds__(PG_THREADS, NT == 2 ? 2 : Q8 ? 4 : 3)
attention_pages_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_k16,
                       const __grid_constant__ CUtensorMap map_v16, const float* __restrict__ ksc, const float* __restrict__ vsc, const bf16* __restrict__ q,
                       int q_stride, const int* __restrict__ block_table, int max_pages, int n_pages, const int* __restrict__ token_pos,
                       const int* __restrict__ token_seq, const PgPlan plan, float* __restrict__ part_acc, float* __restrict__ part_ml, bf16* __restrict__ out,
                       int own_splits, int pre_splits, int nh, int nkv, int page_size, int span, float scale_log2e, int* __restrict__ err) {
    using R = PgRing<D, Q8, NT>;
    constexpr int KS = D / 16, STAGES = R::STAGES, TILE = R::TILE;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * STAGES];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned base = (tc_smem_u32(smem_raw) + 1023u) & ~1023u, scales = base + STAGES * 2 * TILE;
    unsigned char* gbase = smem_raw + (base - tc_smem_u32(smem_raw));
    const unsigned full0 = tc_smem_u32(bars), empty0 = full0 + 8 * STAGES;
    if (tid == 0) {
        for (int i = 0; i < STAGES; i++) {
            mbar_init(full0 + 8 * i, 1);
            mbar_init(empty0 + 8 * i, PG_CONSUMERS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    // Behind wide tiles this kernel needs nothing of theirs, and what comes before them is through when they let it start (attention_tiles.cu): it runs beside
    // them and waits for them at its end, for the sake of what follows both.
    const bool beside = plan.start && plan.n_tiles == 0;
    if (beside) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    else pdl_grid_sync();

    // ---- which rows and keys
    // the blocks of one (prefix tile or token, kv head) follow one another, then come the other kv heads, whose rows lie in the same pages
    const int G = nh / nkv, slots = own_splits + pre_splits, own0 = plan.n_tiles * nkv * pre_splits;
    const bool prefix = (int)blockIdx.x < own0;
    const int n_splits = prefix ? pre_splits : own_splits, at = (int)blockIdx.x - (prefix ? 0 : own0), split = at % n_splits, hk = at / n_splits % nkv, item = at / n_splits / nkv;
    int t = 0, first = 0, count = 1, p, lo = 0;
    if (prefix) {
        const int4 tile = plan.tiles[item];
        first = item * plan.per_tile;
        count = min(tile.x, plan.per_tile);
        p = tile.y - 1;
        if (count <= 0 || p < 0) return;
        t = plan.members[first];
    } else {
        t = item;
        p = token_pos[t];
        lo = p < 0 ? 0 : first_visible(p, span);
        if (plan.start) lo = max(lo, plan.start[t]);
    }
    const int rows = count * G;
    auto row_head = [&](int r) -> size_t {      // of a row below `rows`: which row of [T, nh]
        const int tok = prefix ? plan.members[first + r / G] : t;
        return (size_t)tok * nh + hk * G + r % G;
    };
    const int last = last_in_table(max_pages, page_size);
    if (p > last && tid == 0) atomicExch(err, PG_ERR_PAGE);
    const int tile_lo = lo / PG_BN, n_tiles = p < lo ? 0 : min(p, last) / PG_BN - tile_lo + 1;
    const int n_my = n_tiles > split ? (n_tiles - split + n_splits - 1) / n_splits : 0;
    const int slot = prefix ? own_splits + split : split;
    if (part_acc && n_my == 0) {
        if (tid < rows) *reinterpret_cast<float2*>(part_ml + (row_head(tid) * slots + slot) * 2) = make_float2(-INFINITY, 0.f);
        if (beside) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }

    if (warp == PG_CONSUMERS) {
        // ---- producer.  A page that the sequence does not hold is reported and another one read in its place.
        if (lane == 0) {
            const int* bt = block_table + (size_t)token_seq[t] * max_pages;
            for (int i = 0; i < n_my; i++) {
                const int s = i % STAGES;
                if (i >= STAGES && !mbar_wait(empty0 + 8 * s, ((i / STAGES) - 1) & 1, err, TC_ERR_TIMEOUT_DECODE)) break;
                const int key0 = (tile_lo + split + i * n_splits) * PG_BN;
                int page = key0 / page_size < max_pages ? bt[key0 / page_size] : -1;
                if (page < 0 || page >= n_pages) {
                    atomicExch(err, PG_ERR_PAGE);
                    page = 0;
                }
                const int row = (page * nkv + hk) * page_size + key0 % page_size;
                const unsigned kdst = base + (unsigned)s * 2 * TILE, vdst = kdst + TILE, bar = full0 + 8 * s;
                const int groups = min(PG_BN / 16, (p - key0) / 16 + 1);       // of 16 keys, as many as hold a visible one
                mbar_expect_tx(bar, (unsigned)groups * (2 * TILE / (PG_BN / 16)) + (unsigned)R::SCALES);
                if (Q8) {
                    rows_bulk(scales + s * R::SCALES, ksc + row, PG_BN * 4, bar);
                    rows_bulk(scales + s * R::SCALES + PG_BN * 4, vsc + row, PG_BN * 4, bar);
                }
#pragma unroll
                for (int hx = 0; hx < (Q8 ? 1 : D / 64); hx++) {
                    const int box = hx * (PG_BN * 128), line = Q8 ? D : 128;
                    if (groups == PG_BN / 16) {
                        tma_load_2d(kdst + box, &map_k, hx * 64, row, bar);
                        tma_load_2d(vdst + box, &map_v, hx * 64, row, bar);
                    } else {
                        for (int u = 0; u < groups; u++) {
                            tma_load_2d(kdst + box + u * 16 * line, &map_k16, hx * 64, row + u * 16, bar);
                            tma_load_2d(vdst + box + u * 16 * line, &map_v16, hx * 64, row + u * 16, bar);
                        }
                    }
                }
            }
        }
        __syncwarp();
        if (!part_acc && n_splits > 1) {        // the cluster's two meetings, at the end
            rows_cluster_sync();
            rows_cluster_sync();
        }
        return;
    }

    // ---- consumers: warp w owns keys 16w .. 16w+15 of every tile.  Keys (and channels of the values) are the 16 rows of a product, queries its
    // 8 columns, NT times.
    const int g = lane >> 2, t4 = lane & 3, mtx = lane >> 3;
    // The queries as fragments of column g.  With eight bits a thread's four elements of 16 are neighbours (4 t4 ..), as the bytes of the keys come;
    // any order of the summed index is as good as another.
    unsigned qf[NT][KS][2];
    float row_scale[NT][2];             // of the thread's columns 2 t4 and 2 t4 + 1 of the scores
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int r = nt * 8 + g;
        const bool ok = r < rows;
        const size_t head = ok ? row_head(r) : 0;
        const bf16* src = q + (head / nh) * (size_t)q_stride + (head % nh) * D;
        uint2 raw[KS];
#pragma unroll
        for (int k = 0; k < KS; k++) {
            raw[k] = make_uint2(0u, 0u);
            if (!ok) continue;
            if (Q8) {
                raw[k] = *reinterpret_cast<const uint2*>(src + k * 16 + t4 * 4);
            } else {
                raw[k].x = *reinterpret_cast<const unsigned*>(src + k * 16 + t4 * 2);
                raw[k].y = *reinterpret_cast<const unsigned*>(src + k * 16 + 8 + t4 * 2);
            }
        }
        float down = 1.f;
        if (Q8) {
            unsigned top = 0;           // the largest magnitude's bits
#pragma unroll
            for (int k = 0; k < KS; k++)
                top = max(max(top, max(raw[k].x & 0x7fffu, (raw[k].x >> 16) & 0x7fffu)), max(raw[k].y & 0x7fffu, (raw[k].y >> 16) & 0x7fffu));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // a power of two that brings the largest to [2^10, 2^11): 128 products with 127 stay below 2^25
            const int ex = max((int)(top >> 7) - 127, -116);
            const float up = __int_as_float((10 - ex + 127) << 23);
            down = __int_as_float((ex - 10 + 127) << 23);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                qf[nt][k][0] = pg_half2(__uint_as_float(raw[k].x << 16) * up, __uint_as_float(raw[k].x & 0xffff0000u) * up);
                qf[nt][k][1] = pg_half2(__uint_as_float(raw[k].y << 16) * up, __uint_as_float(raw[k].y & 0xffff0000u) * up);
            }
        } else {
#pragma unroll
            for (int k = 0; k < KS; k++) {
                qf[nt][k][0] = raw[k].x;
                qf[nt][k][1] = raw[k].y;
            }
        }
        row_scale[nt][0] = scale_log2e * __shfl_sync(0xffffffffu, down, t4 * 8);
        row_scale[nt][1] = scale_log2e * __shfl_sync(0xffffffffu, down, t4 * 8 + 4);
    }

    // Per column: m, what the sums l are relative to, and mv, what the accumulators are (m itself for bfloat16 rows); both follow the largest score
    // only once it is 2^8 ahead, which a vote finds, so that the maxima cost no shuffles otherwise.  A weight is at most 2^8 that way.
    float m[NT][2], mv[NT][2], l[NT][2], o[NT][KS][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        m[nt][0] = m[nt][1] = mv[nt][0] = mv[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; i++) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    }

    for (int i = 0; i < n_my; i++) {
        const int s = i % STAGES;
        if (!__all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, (i / STAGES) & 1, err, TC_ERR_TIMEOUT_DECODE))) break;
        const int key0 = (tile_lo + split + i * n_splits) * PG_BN + warp * 16;
        if (key0 <= p && key0 + 15 >= lo) {
            const unsigned kbase = base + (unsigned)s * 2 * TILE, vbase = kbase + TILE;
            float sc[NT][4], sv[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) sc[nt][e] = sv[nt][e] = 0.f;
            const int krow = warp * 16 + (mtx & 1) * 8 + (lane & 7);
            if (Q8) {
#pragma unroll
                for (int k = 0; k < KS; k += 2) {
                    unsigned b[4];
                    pg_ldm(b, kbase + pg_off<D, Q8>(krow, k + (mtx >> 1)));
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const unsigned a[4] = {pg_widen(b[2 * u], 0x4140), pg_widen(b[2 * u + 1], 0x4140), pg_widen(b[2 * u], 0x4342), pg_widen(b[2 * u + 1], 0x4342)};
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) pg_mma<true>(u ? sv[nt] : sc[nt], a, qf[nt][k + u][0], qf[nt][k + u][1]);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    unsigned a[4];
                    pg_ldm(a, kbase + pg_off<D, Q8>(krow, k * 2 + (mtx >> 1)));
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) pg_mma<false>(k & 1 ? sv[nt] : sc[nt], a, qf[nt][k][0], qf[nt][k][1]);
                }
            }
            // scores in units of log2: element e of a thread is key g + 8 (e / 2), column 2 t4 + e % 2
            float lv[2] = {0.f, 0.f}, kf[2] = {1.f, 1.f};       // log2 of the values' scales, the keys' scales
            if (Q8) {
                const unsigned at = scales + s * R::SCALES + (warp * 16 + g) * 4;
                float v[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(kf[e]) : "r"(at + e * 32));
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[e]) : "r"(at + e * 32 + PG_BN * 4));
                    lv[e] = pg_log2(v[e]);
                }
            }
            const bool edge = key0 + 15 > p || key0 < lo;
            bool over = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float v = (sc[nt][e] + sv[nt][e]) * row_scale[nt][e & 1];
                    if (Q8) v *= kf[e >> 1];
                    float w = v + lv[e >> 1];
                    if (edge) {
                        const int key = key0 + g + (e >> 1) * 8;
                        if (key > p || key < lo) v = w = -INFINITY;
                    }
                    sc[nt][e] = v;
                    sv[nt][e] = w;
                    over |= v > m[nt][e & 1] + PG_AHEAD;
                    if (Q8) over |= w > mv[nt][e & 1] + PG_AHEAD;
                }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float top = fmaxf(sc[nt][e], sc[nt][e + 2]), topv = fmaxf(sv[nt][e], sv[nt][e + 2]);
#pragma unroll
                        for (int k = 4; k < 32; k *= 2) {
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
                            if (Q8) topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, k));
                        }
                        top = fmaxf(top, m[nt][e]);
                        topv = Q8 ? fmaxf(topv, mv[nt][e]) : top;
                        l[nt][e] *= top == -INFINITY ? 1.f : fast_exp2(m[nt][e] - top);
                        const float keep = topv == -INFINITY ? 1.f : fast_exp2(mv[nt][e] - topv);
                        m[nt][e] = top;
                        mv[nt][e] = topv;
#pragma unroll
                        for (int c = 0; c < KS; c++) {
                            o[nt][c][e] *= keep;
                            o[nt][c][e + 2] *= keep;
                        }
                    }
            }
            unsigned pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float pw[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float ref = m[nt][e & 1], refv = mv[nt][e & 1];
                    const float pe = fast_exp2(sc[nt][e] - (ref == -INFINITY ? 0.f : ref));
                    l[nt][e & 1] += pe;
                    pw[e] = Q8 ? fast_exp2(sv[nt][e] - (refv == -INFINITY ? 0.f : refv)) : pe;
                }
                pf[nt][0] = pg_transpose(Q8 ? pg_half2(pw[0], pw[1]) : pg_bf162(pw[0], pw[1]));
                pf[nt][1] = pg_transpose(Q8 ? pg_half2(pw[2], pw[3]) : pg_bf162(pw[2], pw[3]));
            }
            if (Q8) {
#pragma unroll
                for (int c = 0; c < KS; c += 2) {
                    unsigned b[4];
                    pg_ldm_t(b, vbase + pg_off<D, Q8>(krow, c + (mtx >> 1)));
#pragma unroll
                    for (int u = 0; u < 2; u++) {           // rows n and n + 8: channels 16 (c + u) + 2 n and + 2 n + 1
                        const unsigned a[4] = {pg_widen(b[2 * u], 0x4240), pg_widen(b[2 * u], 0x4341), pg_widen(b[2 * u + 1], 0x4240), pg_widen(b[2 * u + 1], 0x4341)};
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) pg_mma<true>(o[nt][c + u], a, pf[nt][0], pf[nt][1]);
                    }
                }
            } else {
                if (edge) {
                    // rows of hidden keys may hold anything, and 0 x NaN would not be 0
                    unsigned char* v = gbase + (size_t)s * 2 * TILE + TILE;
                    for (int j = lane; j < 16 * 2 * KS; j += 32) {
                        const int r = j / (2 * KS), c = j % (2 * KS);
                        if (key0 + r > p || key0 + r < lo) *reinterpret_cast<uint4*>(v + pg_off<D, Q8>(warp * 16 + r, c)) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // before the stage is filled again
                    __syncwarp();
                }
                const int vrow = warp * 16 + (mtx >> 1) * 8 + (lane & 7);
#pragma unroll
                for (int c = 0; c < KS; c++) {
                    unsigned a[4];
                    pg_ldm_t(a, vbase + pg_off<D, Q8>(vrow, c * 2 + (mtx & 1)));
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) pg_mma<false>(o[nt][c], a, pf[nt][0], pf[nt][1]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(empty0 + 8 * s) : "memory");
    }

    // ---- join the warps (ascending) through the ring's memory: every load has landed and been read
    asm volatile("bar.sync 1, %0;" ::"n"(PG_CONSUMERS * 32) : "memory");
    float* joined = reinterpret_cast<float*>(gbase);            // [PG_CONSUMERS][16][D + 4]: accumulators, m, l, mv
    constexpr int ROW = D + 4;
    static_assert((PG_CONSUMERS + 1) * 16 * ROW * 4 <= STAGES * 2 * TILE, "the joined rows and the share must fit the ring");
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
            for (int k = 4; k < 32; k *= 2) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], k);
            const int r = nt * 8 + t4 * 2 + e;
            if (r >= rows) continue;
            float* dst = joined + ((size_t)warp * 16 + r) * ROW;
#pragma unroll
            for (int c = 0; c < KS; c++) {
                if (Q8) {
                    *reinterpret_cast<float2*>(dst + c * 16 + g * 2) = make_float2(o[nt][c][e], o[nt][c][e + 2]);
                } else {
                    dst[c * 16 + g] = o[nt][c][e];
                    dst[c * 16 + 8 + g] = o[nt][c][e + 2];
                }
            }
            if (g == 0) *reinterpret_cast<float4*>(dst + D) = make_float4(m[nt][e], l[nt][e], mv[nt][e], 0.f);
        }
    asm volatile("bar.sync 1, %0;" ::"n"(PG_CONSUMERS * 32) : "memory");
    // the block's share of every row: accumulators relative to m, m and l; a row without keys has l = 0.  A thread makes four channels (one by one the
    // warps' factors cost more than the sums: 16 rows behind a common prefix of 128 positions 13.1 us).
    float* share = joined + (size_t)PG_CONSUMERS * 16 * ROW;        // [16][ROW]
    const bool alone = !part_acc && n_splits == 1;
    for (int idx = tid; idx < rows * (D / 4); idx += PG_CONSUMERS * 32) {
        const int r = idx / (D / 4), c = (idx - r * (D / 4)) * 4;
        float4 w[PG_CONSUMERS], v[PG_CONSUMERS];
        float M = -INFINITY;
#pragma unroll
        for (int k = 0; k < PG_CONSUMERS; k++) {
            w[k] = *reinterpret_cast<const float4*>(joined + ((size_t)k * 16 + r) * ROW + D);
            v[k] = *reinterpret_cast<const float4*>(joined + ((size_t)k * 16 + r) * ROW + c);
            M = fmaxf(M, w[k].x);
        }
        const float ref = M == -INFINITY ? 0.f : M;
        float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f;
#pragma unroll
        for (int k = 0; k < PG_CONSUMERS; k++) {
            if (w[k].y == 0.f) continue;                        // no visible keys; a sum that is no number goes on
            pg_add(num, v[k], w[k].z == -INFINITY ? 1.f : fast_exp2(w[k].z - ref));
            den += w[k].y * (w[k].x == -INFINITY ? 1.f : fast_exp2(w[k].x - ref));
        }
        if (alone) {
            pg_result(out + row_head(r) * D + c, num, den);
        } else if (part_acc) {
            const size_t at = row_head(r) * slots + slot;
            *reinterpret_cast<float4*>(part_acc + at * D + c) = num;
            if (c == 0) *reinterpret_cast<float2*>(part_ml + at * 2) = make_float2(M, den);
        } else {
            *reinterpret_cast<float4*>(share + r * ROW + c) = num;
            if (c == 0) *reinterpret_cast<float2*>(share + r * ROW + D) = make_float2(M, den);
        }
    }
    if (beside) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (alone || part_acc) return;
    // ---- join the cluster's shares (ascending): every block writes a part of the rows
    rows_cluster_sync();
    const unsigned share_at = tc_smem_u32(share);
    for (int idx = split * (PG_CONSUMERS * 32) + tid; idx < rows * (D / 4); idx += n_splits * (PG_CONSUMERS * 32)) {
        const int r = idx / (D / 4), c = (idx - r * (D / 4)) * 4;
        const unsigned row_at = share_at + r * ROW * 4;
        float4 v[PG_MAX_CLUSTER], num = make_float4(0.f, 0.f, 0.f, 0.f);
        float2 ml[PG_MAX_CLUSTER];
        float M = -INFINITY, den = 0.f;
#pragma unroll
        for (int k = 0; k < PG_MAX_CLUSTER; k++) {
            ml[k] = k < n_splits ? pg_remote2(row_at + D * 4, k) : make_float2(-INFINITY, 0.f);
            v[k] = k < n_splits ? rows_remote4(row_at + c * 4, k) : make_float4(0.f, 0.f, 0.f, 0.f);
            M = fmaxf(M, ml[k].x);
        }
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int k = 0; k < PG_MAX_CLUSTER; k++) {
            if (k >= n_splits || ml[k].y == 0.f) continue;
            const float f = ml[k].x == -INFINITY ? 1.f : fast_exp2(ml[k].x - ref);
            pg_add(num, v[k], f);
            den += f * ml[k].y;
        }
        pg_result(out + row_head(r) * D + c, num, den);
    }
    rows_cluster_sync();              // the others may still read this block's shares
}

// out[t, h] = sum over the shares (ascending) of acc 2^(m - M) / sum of l 2^(m - M): a token's own and, where it has a prefix in common with
// others, the prefix's.  A share without keys has l = 0 and no accumulators; a token without any gets zeros.
template <int D>
__global__ void __launch_bounds__(D)
attention_pages_join_kernel(const float* __restrict__ part_acc, const float* __restrict__ part_ml, bf16* __restrict__ out, int own_splits, int pre_splits,
                            const int* __restrict__ start, int nh) {
    pdl_grid_sync();
    const int h = blockIdx.x, t = blockIdx.y, c = threadIdx.x, lane = threadIdx.x & 31, slots = own_splits + pre_splits;
    const int n = start && start[t] > 0 ? slots : own_splits;
    const size_t o = ((size_t)t * nh + h) * slots;
    float2 ml[2];           // share `lane` and share 32 + `lane`
#pragma unroll
    for (int k = 0; k < 2; k++) ml[k] = lane + 32 * k < n ? *reinterpret_cast<const float2*>(part_ml + (o + lane + 32 * k) * 2) : make_float2(-INFINITY, 0.f);
    const float M = warp_max(fmaxf(ml[0].x, ml[1].x)), ref = M == -INFINITY ? 0.f : M;
    float w[2];
#pragma unroll
    for (int k = 0; k < 2; k++) w[k] = ml[k].y == 0.f ? 0.f : ml[k].x == -INFINITY ? 1.f : fast_exp2(ml[k].x - ref);
    float num = 0.f, den = 0.f;
    for (int s0 = 0; s0 < n; s0 += 8) {
        float v[8], f[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int s = s0 + k;
            f[k] = __shfl_sync(0xffffffffu, s < 32 ? w[0] : w[1], s & 31);
            const float l = __shfl_sync(0xffffffffu, s < 32 ? ml[0].y : ml[1].y, s & 31);
            if (f[k] != 0.f) den += f[k] * l;
            v[k] = s < n && f[k] != 0.f ? part_acc[(o + s) * D + c] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; k++) num += f[k] * v[k];
    }
    out[((size_t)t * nh + h) * D + c] = __float2bfloat16_rn(den == 0.f ? 0.f : num / den);
}

// ---- host side

template <int D, bool Q8>
static int pg_launch(const void* q, int q_stride, const void* kc, const void* vc, const float* ksc, const float* vsc, long long n_pages, const int* block_table, int max_pages,
                     const int* token_pos, const int* token_seq, const PgPlan& plan, float* part_acc, float* part_ml, void* out, int T, int nh, int nkv, int page_size,
                     int span, float scale, int own_splits, int pre_splits, int* err, cudaStream_t s) {
    CUtensorMap mk, mv, mk16, mv16;
    const long long rows = n_pages * nkv * page_size;
    const CUtensorMapSwizzle swizzle = Q8 && D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    int rc;
    if ((rc = rows_make_map(&mk, kc, rows, D, PG_BN, Q8, swizzle)) || (rc = rows_make_map(&mv, vc, rows, D, PG_BN, Q8, swizzle)) || (rc = rows_make_map(&mk16, kc, rows, D, 16, Q8, swizzle)) ||
        (rc = rows_make_map(&mv16, vc, rows, D, 16, Q8, swizzle)))
        return rc;
    // eight rows in a block's products where no block has more
    const bool eight = nh / nkv * (plan.n_tiles ? plan.per_tile : 1) <= 8;
    auto kern = eight ? attention_pages_kernel<D, Q8, 1> : attention_pages_kernel<D, Q8, 2>;
    const int smem = eight ? PgRing<D, Q8, 1>::BYTES : PgRing<D, Q8, 2>::BYTES;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    const bool shares = part_acc != nullptr;
    const long long blocks = (long long)nkv * ((long long)plan.n_tiles * pre_splits + (long long)T * own_splits);
    if (blocks > 0x7fffffffLL) return ILLM_ERR_BAD_ARG;
    rc = illm_launch_cluster(kern, dim3((unsigned)blocks), dim3(PG_THREADS), shares ? 1 : own_splits, smem, s, mk, mv, mk16,
                             mv16, ksc, vsc, (const bf16*)q, q_stride, block_table, max_pages, (int)n_pages, token_pos, token_seq, plan, part_acc, part_ml, (bf16*)out,
                             own_splits, pre_splits, nh, nkv, page_size, span, scale * 1.4426950408889634f, err);
    if (rc || !shares) return rc;
    illm_launch(attention_pages_join_kernel<D>, dim3(nh, T), dim3(D), 0, s, (const float*)part_acc, (const float*)part_ml, (bf16*)out, own_splits, pre_splits,
                plan.start, nh);
    return illm_launch_status();
}

// Single tokens: q, rows of q_stride bfloat16 elements whose first nh * d are the query heads; kc, vc one entry's pages
// [n_pages, nkv, page_size, d] of bytes with their scales ksc, vsc, or (ksc, vsc nullptr) of bfloat16; page_size a multiple of 64, d 64
// or 128, at most 16 query heads per kv head.  plan_start nullptr, or a plan (PgPlan; then span 0): its n_tiles tiles, of at most per_tile members and 16 rows (members times nh / nkv),
// are walked here; with n_tiles 0
// their pre_splits shares are what the launch before this one makes, which has to be illm_attention_tiles_prefix's (slot0 = own_splits): the two run side by side.  own_splits, pre_splits: at most 32 each,
// pre_splits 0 without a plan.  Scratch: part_acc float [T, nh, slots, d], part_ml float [T, nh, slots, 2], or, without a plan and with up to 8 splits,
// nullptr: then the blocks of a (token, kv head) are a cluster and there is no second kernel.  That is the faster way while the blocks find room together (one
// sequence of 8 kv heads at 1,777 keys 6.6 us and 7.3), and the slower one where they have to wait for one another's places (64 sequences of 32 kv heads at 300
// keys in two parts 57 us and 47).  err: 7 a wait ran out, 8 a visible position without a page.
extern "C" int illm_attention_pages(const void* q, int q_stride, const void* kc, const void* vc, const float* ksc, const float* vsc, long long n_pages,
                                    const int* block_table, int max_pages, const int* token_pos, const int* token_seq, const int* plan_start, const int* plan_tiles,
                                    const int* plan_members, int n_tiles, int per_tile, float* part_acc, float* part_ml, void* out, int T, int nh, int nkv, int d, int page_size,
                                    int span, float scale, int own_splits, int pre_splits, int* err, void* stream) {
    if (T <= 0) return 0;
    if (nkv <= 0 || nh <= 0 || nh % nkv || nh / nkv > 16 || T > 65535 || nkv > 65535 || n_tiles < 0 || n_tiles > 65535 || (q_stride & 7) || page_size <= 0 ||
        page_size % PG_BN || max_pages <= 0 || n_pages <= 0 || n_pages * nkv * page_size > 0x7fffffffLL || own_splits < 1 || own_splits > PG_MAX_SPLITS || pre_splits < 0 ||
        pre_splits > PG_MAX_SPLITS || !q || ((uintptr_t)q & 15) || !kc || !vc || ((uintptr_t)kc & 15) || ((uintptr_t)vc & 15) || (!ksc) != (!vsc) || ((uintptr_t)ksc & 15) ||
        ((uintptr_t)vsc & 15) || !err || (plan_start && (span != 0 || pre_splits < 1)) || (!plan_start && (n_tiles > 0 || pre_splits != 0)) ||
        (n_tiles > 0 && (per_tile < 1 || per_tile > 16 || per_tile * (nh / nkv) > 16 || !plan_tiles || !plan_members || ((uintptr_t)plan_tiles & 15))) || ((own_splits > PG_MAX_CLUSTER || plan_start) && !part_acc) || (!part_acc) != (!part_ml) || ((uintptr_t)part_ml & 7) || !out || !token_pos || !token_seq || !block_table)
        return ILLM_ERR_BAD_ARG;
    const PgPlan plan = {plan_start, reinterpret_cast<const int4*>(plan_tiles), plan_members, n_tiles, per_tile};
    cudaStream_t s = (cudaStream_t)stream;
#define PG_CASE(DD, QQ)                                                                                                                                        \
    if (d == DD && (ksc != nullptr) == QQ)                                                                                                                     \
        return pg_launch<DD, QQ>(q, q_stride, kc, vc, ksc, vsc, n_pages, block_table, max_pages, token_pos, token_seq, plan, part_acc, part_ml, out, T, nh, nkv, \
                                 page_size, span, scale, own_splits, pre_splits, err, s);
    PG_CASE(128, true) PG_CASE(64, true) PG_CASE(128, false) PG_CASE(64, false)
#undef PG_CASE
    return ILLM_ERR_BAD_ARG;
}
