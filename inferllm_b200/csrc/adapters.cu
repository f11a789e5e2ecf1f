// Low-rank adapters of many requests beside a shared projection:
//   y[t] = x[t] W^T + s_a (x[t] A_a^T) B_a^T,   a the adapter of token t's request, or none.
// x [T, K], W [N, K]; the adapters of a projection lie in one piece: A [count, R, K] and B [count, R / 16, N, 16] (the second
// factor by groups of 16 ranks, so that one K step of a tensor-core product, or 32 to 64 bytes of one output, lie together),
// R the largest rank rounded up to 16, rows beyond an adapter's own rank zero and, where they fill a group, never read.
// Which token has which adapter comes as a plan (adapters.h).
//
// The general form (both types): the shared product by the package's own kernels into float32, then
//   shrink   v[t] = s_a x[t] A_a^T: a block per 8 tokens of the plan's order and rank group, a warp per two ranks, which
//            reads a row of A once for the tokens of a slot;
//   expand   y[t, n] = base[t, n] + v[t] . B_a[n]: a thread per output column, the slot's 16 values of B in registers.
// Sums are float32 in one order per token, whatever else is in the batch.
#include "adapters.h"
#include "common.cuh"
#include "kernels.h"

#define AD_TOKENS 8
#define AD_COLS 128

struct AdPlan {
    const int *counts, *token_adapter, *order, *slot_begin, *slot_adapter, *slot_group, *groups, *tile_chunk, *chunk_tile, *chunk_groups;
};
static AdPlan ad_plan(const int* plan, const AdapterPlanSizes& s) {
    const AdapterPlanLayout l = adapter_plan_layout(s);
    return AdPlan{plan + l.counts, plan + l.token_adapter, plan + l.order, plan + l.slot_begin, plan + l.slot_adapter, plan + l.slot_group, plan + l.groups,
                  plan + l.tile_chunk, plan + l.chunk_tile, plan + l.chunk_groups};
}

// v[t, 16 g + r] for the ranks of group g of token t's adapter, float32 [T, R]
template <typename T>
__global__ void __launch_bounds__(256)
adapter_shrink_kernel(const T* __restrict__ x, int K, const T* __restrict__ a, const float* __restrict__ scales, int R, const AdPlan plan, int tokens,
                      float* __restrict__ v) {
    pdl_grid_sync();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = blockIdx.y;
    const int n_slots = plan.counts[0], p0 = blockIdx.x * AD_TOKENS, p1 = min(tokens, p0 + AD_TOKENS);
    int slot = 0;
    for (int p = p0; p < p1;) {
        while (slot < n_slots && plan.slot_begin[slot + 1] <= p) slot++;
        if (slot >= n_slots) return;                    // the rest has no adapter
        const int e = min(p1, plan.slot_begin[slot + 1]), n = e - p;
        if (g < plan.slot_group[slot + 1] - plan.slot_group[slot]) {
            const int ad = plan.slot_adapter[slot];
            const T* a0 = a + ((long long)ad * R + g * ADAPTER_GROUP + warp * 2) * K;
            const T* xr[AD_TOKENS];
            float acc[2][AD_TOKENS];
#pragma unroll
            for (int i = 0; i < AD_TOKENS; i++) {
                xr[i] = x + (long long)plan.order[p + min(i, n - 1)] * K;
                acc[0][i] = acc[1][i] = 0.f;
            }
            for (int k = lane; k < K; k += 32) {
                const float w0 = to_f32(a0[k]), w1 = to_f32(a0[K + k]);
#pragma unroll
                for (int i = 0; i < AD_TOKENS; i++) {
                    const float xv = to_f32(xr[i][k]);
                    acc[0][i] = fmaf(xv, w0, acc[0][i]);
                    acc[1][i] = fmaf(xv, w1, acc[1][i]);
                }
            }
#pragma unroll
            for (int i = 0; i < AD_TOKENS; i++) {
                acc[0][i] = warp_sum(acc[0][i]);
                acc[1][i] = warp_sum(acc[1][i]);
            }
            const float s = scales[ad];
            if (lane == 0)
#pragma unroll
                for (int i = 0; i < AD_TOKENS; i++)
                    if (i < n) {
                        float* to = v + (long long)plan.order[p + i] * R + g * ADAPTER_GROUP + warp * 2;
                        to[0] = s * acc[0][i];
                        to[1] = s * acc[1][i];
                    }
        }
        p = e;
    }
}

template <typename T, typename TOut>
__global__ void __launch_bounds__(AD_COLS)
adapter_expand_kernel(const float* base, int N, const T* __restrict__ b, const float* __restrict__ v, int R, const AdPlan plan, int tokens, TOut* out) {
    pdl_grid_sync();
    const int col = blockIdx.x * AD_COLS + threadIdx.x;
    const int n_slots = plan.counts[0], p0 = blockIdx.y * AD_TOKENS, p1 = min(tokens, p0 + AD_TOKENS);
    if (col >= N) return;
    int slot = 0;
    for (int p = p0; p < p1;) {
        while (slot < n_slots && plan.slot_begin[slot + 1] <= p) slot++;
        const int e = slot < n_slots ? min(p1, plan.slot_begin[slot + 1]) : p1, n = e - p;
        float acc[AD_TOKENS];
        for (int i = 0; i < AD_TOKENS; i++) acc[i] = 0.f;
        if (slot < n_slots) {
            const int ad = plan.slot_adapter[slot], n_g = plan.slot_group[slot + 1] - plan.slot_group[slot];
            for (int g = 0; g < n_g; g++) {
                float w[ADAPTER_GROUP];
                const T* bw = b + (((long long)ad * (R / ADAPTER_GROUP) + g) * N + col) * ADAPTER_GROUP;
                load8(bw, w);
                load8(bw + 8, w + 8);
#pragma unroll
                for (int i = 0; i < AD_TOKENS; i++)
                    if (i < n) {
                        const float* vt = v + (long long)plan.order[p + i] * R + g * ADAPTER_GROUP;
#pragma unroll
                        for (int r = 0; r < ADAPTER_GROUP; r++) acc[i] = fmaf(vt[r], w[r], acc[i]);
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < AD_TOKENS; i++)
            if (i < n) {
                const long long at = (long long)plan.order[p + i] * N + col;
                out[at] = from_f32<TOut>(base[at] + acc[i]);
            }
        p = e;
    }
}

// Bytes of workspace that illm_linear_adapters needs.
extern "C" long long illm_linear_adapters_ws(int dtype, int T, int N, int K, int R, int groups, int chunks) {
    const long long v = (long long)T * R * 4, base = dtype == ILLM_BF16 ? (long long)T * N * 4 : 0;
    return (v + 255) / 256 * 256 + base;
}

template <typename TX, typename TOut>
static int ad_general(const void* x, const void* w, int T, int N, int K, const void* a, const void* b, const float* scales, int R, const AdapterPlanSizes& sz,
                      const int* plan_dev, TOut* out, char* ws, int* err, cudaStream_t s) {
    const AdPlan plan = ad_plan(plan_dev, sz);
    float* v = (float*)ws;
    const int groups = R / ADAPTER_GROUP, tiles = (T + AD_TOKENS - 1) / AD_TOKENS;
    float* base;
    int rc;
    if (sizeof(TX) == 4) {
        base = (float*)out;
        rc = illm_gemm_f32_nt((const float*)x, (const float*)w, base, T, N, K, K, K, N, err, s);
    } else {
        base = (float*)(ws + ((size_t)T * R * 4 + 255) / 256 * 256);
        rc = T <= 64 ? illm_gemm_bf16_tc(x, w, base, ILLM_F32, T, N, K, nullptr, 1, err, s, 0) : illm_gemm_bf16_tc2(x, w, base, ILLM_F32, 0, T, N, K, err, s);
    }
    if (rc != 0) return rc;
    if (sz.slots > 0)
        illm_launch(adapter_shrink_kernel<TX>, dim3(tiles, groups), dim3(256), 0, s, (const TX*)x, K, (const TX*)a, scales, R, plan, T, v);
    illm_launch(adapter_expand_kernel<TX, TOut>, dim3((N + AD_COLS - 1) / AD_COLS, tiles), dim3(AD_COLS), 0, s, (const float*)base, N, (const TX*)b,
                (const float*)v, R, plan, T, out);
    return illm_launch_status();
}

// out [T, N] = x W^T + the tokens' adapters.  dtype: of x, W, A and B; out_dtype float32 or that.  plan: the device array laid
// out by adapter_plan_layout({T, slots, groups, chunks}).  ws: illm_linear_adapters_ws bytes, 256-byte aligned.
extern "C" int illm_linear_adapters(const void* x, const void* w, int dtype, int T, int N, int K, const void* a, const void* b, const float* scales,
                                    int count, int R, const int* plan, int slots, int groups, int chunks, void* out, int out_dtype, void* ws, int* err,
                                    void* stream) {
    if (T <= 0 || N <= 0) return 0;
    if (K <= 0 || count <= 0 || R <= 0 || R % ADAPTER_GROUP || R > ADAPTER_GROUP * ADAPTER_MAX_GROUPS || slots < 0 || groups < 0 || chunks < 0 || !ws || !plan ||
        T > 65535 * AD_TOKENS)
        return ILLM_ERR_BAD_ARG;
    if (dtype == ILLM_BF16 && ((K & 7) || ((uintptr_t)x & 15) || ((uintptr_t)w & 15) || ((uintptr_t)a & 15) || ((uintptr_t)b & 15))) return ILLM_ERR_BAD_ARG;
    const AdapterPlanSizes sz{T, slots, groups, chunks};
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == ILLM_F32 && out_dtype == ILLM_F32)
        return ad_general<float, float>(x, w, T, N, K, a, b, scales, R, sz, plan, (float*)out, (char*)ws, err, s);
    if (dtype == ILLM_BF16 && out_dtype == ILLM_BF16)
        return ad_general<bf16, bf16>(x, w, T, N, K, a, b, scales, R, sz, plan, (bf16*)out, (char*)ws, err, s);
    if (dtype == ILLM_BF16 && out_dtype == ILLM_F32)
        return ad_general<bf16, float>(x, w, T, N, K, a, b, scales, R, sz, plan, (float*)out, (char*)ws, err, s);
    return ILLM_ERR_BAD_ARG;
}
