// Attention of any token over a cache of eight-bit rows (kv_int8.cu): the kernel for head sizes, page sizes and activations that the
// tensor-core kernels (attention_pages.cu, attention_tiles.cu) do not take, among them float32, where it keeps float32 throughout.
//
// o = sum_j p_j s^v_j (u^v_j - 128), p = softmax over the visible j of scale s^k_j sum_c q_c (u^k_jc - 128)
// (src/kern/naive/naive.cpp:576-604, :531-553, :209-240, :634-662).
// A block takes one (token, head).  Its eight warps walk the visible keys 32 at a time: a lane makes the score of one key alone (its
// row in eight-byte pieces, the query from shared memory), the warp agrees on the running maximum, and for the values the lanes
// change roles, a lane for eight channels; what the warps have is added up at the end in ascending order.  A score and a weight
// are float32.  Bound by its loads, which lie a row apart between lanes (a lane's 16 loads of a row of 128 share its four sectors), four of
// them in flight: 8 sequences of up to 4,096 positions with 32 / 32 heads of 128 in float32 223 us, 64 of 2,048 with heads of 96 in bfloat16 400 and one 53 (one load
// at a time 350, 646 and 85; four warps besides 660, 651 and 160; sixteen warps 336, 1,140 and 49).
#include <math.h>

#include "common.cuh"

#define AI_WARPS 8

template <typename TA>
__global__ void __launch_bounds__(AI_WARPS * 32)
attention_int8_kernel(const TA* __restrict__ q, int q_stride, const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc,
                      const float* __restrict__ ksc, const float* __restrict__ vsc, const int* __restrict__ block_table, int max_pages, int n_pages,
                      const int* __restrict__ token_pos, const int* __restrict__ token_seq, TA* __restrict__ out, int nh, int nkv, int d, int page_size, int span,
                      float scale_log2e, int* __restrict__ err) {
    pdl_grid_sync();
    __shared__ float qs[256], merged[AI_WARPS][256], tops[AI_WARPS], sums[AI_WARPS];
    const int t = blockIdx.x, h = blockIdx.y, hk = h / (nh / nkv), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pieces = d >> 3;
    for (int c = threadIdx.x; c < d; c += AI_WARPS * 32) qs[c] = to_f32(q[(size_t)t * q_stride + (size_t)h * d + c]);
    __syncthreads();
    const int place = token_pos[t], p = min(place, last_in_table(max_pages, page_size)), lo = p < 0 ? 0 : min(first_visible(place, span), p + 1);
    if (p < place && threadIdx.x == 0) atomicExch(err, 8);
    const int* bt = block_table + (size_t)token_seq[t] * max_pages;
    float m = -INFINITY, l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j0 = lo + warp * 32; j0 <= p; j0 += AI_WARPS * 32) {
        const int j = j0 + lane;
        long long row = -1;
        if (j <= p) {
            const int page = j / page_size < max_pages ? bt[j / page_size] : -1;
            if (page < 0 || page >= n_pages) atomicExch(err, 8);
            else row = ((long long)page * nkv + hk) * page_size + j % page_size;
        }
        float s = -INFINITY, sv = 0.f;
        if (row >= 0) {
            float dot = 0.f;
            const unsigned char* k = kc + row * d;
#pragma unroll 4
            for (int c = 0; c < pieces; c++) {
                const uint2 w = *reinterpret_cast<const uint2*>(k + c * 8);
#pragma unroll
                for (int i = 0; i < 8; i++) dot = fmaf(qs[c * 8 + i], (float)((int)((i < 4 ? w.x : w.y) >> (8 * (i & 3)) & 255u) - 128), dot);
            }
            s = dot * ksc[row] * scale_log2e;
            sv = vsc[row];
        }
        const float top = fmaxf(m, warp_max(s)), ref = top == -INFINITY ? 0.f : top, keep = exp2f(m - ref);
        const float w = row >= 0 ? exp2f(s - ref) : 0.f, wv = row >= 0 ? w * sv : 0.f;
        l = l * keep + warp_sum(w);
        m = top;
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] *= keep;
        const int n = min(32, p - j0 + 1);
#pragma unroll 4
        for (int i = 0; i < n; i++) {
            const float f = __shfl_sync(0xffffffffu, wv, i);
            const long long r = __shfl_sync(0xffffffffu, row, i);
            const uint2 v = r < 0 || lane >= pieces ? make_uint2(0x80808080u, 0x80808080u) : *reinterpret_cast<const uint2*>(vc + r * d + lane * 8);
#pragma unroll
            for (int k = 0; k < 8; k++) acc[k] = fmaf(f, (float)((int)((k < 4 ? v.x : v.y) >> (8 * (k & 3)) & 255u) - 128), acc[k]);
        }
    }
    if (lane < pieces)
#pragma unroll
        for (int k = 0; k < 8; k++) merged[warp][lane * 8 + k] = acc[k];
    if (lane == 0) {
        tops[warp] = m;
        sums[warp] = l;
    }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < AI_WARPS; w++) top = fmaxf(top, tops[w]);
    const float ref = top == -INFINITY ? 0.f : top;
    for (int c = threadIdx.x; c < d; c += AI_WARPS * 32) {
        float num = 0.f, den = 0.f;
#pragma unroll
        for (int w = 0; w < AI_WARPS; w++) {
            if (sums[w] == 0.f) continue;           // no keys; a sum that is no number goes on
            const float f = tops[w] == -INFINITY ? 1.f : exp2f(tops[w] - ref);
            num += merged[w][c] * f;
            den += sums[w] * f;
        }
        out[((size_t)t * nh + h) * d + c] = from_f32<TA>(den == 0.f ? 0.f : num / den);
    }
}

// q: rows of q_stride elements whose first nh * d are the query heads; out [T, nh d], zeros for a token without visible keys.
// span: see first_visible.  err: 8 a visible position without a page.
extern "C" int illm_attention_int8(const void* q, int q_stride, const void* kc, const void* vc, const float* ksc, const float* vsc, const int* block_table,
                                   int max_pages, long long n_pages, const int* token_pos, const int* token_seq, void* out, int act_dtype, int T, int nh, int nkv,
                                   int d, int page_size, int span, float scale, int* err, void* stream) {
    if (T <= 0) return 0;
    if (nkv <= 0 || nh <= 0 || nh % nkv || nh > 65535 || d <= 0 || d > 256 || (d & 7) || page_size <= 0 || max_pages <= 0 || n_pages <= 0 || n_pages > 0x7fffffffLL ||
        !q || !kc || !vc || !ksc || !vsc || ((uintptr_t)kc & 7) || ((uintptr_t)vc & 7) || !err)
        return ILLM_ERR_BAD_ARG;
    cudaStream_t s = (cudaStream_t)stream;
    const float f = scale * 1.4426950408889634f;
#define AI_RUN(TA)                                                                                                                                      \
    illm_launch(attention_int8_kernel<TA>, dim3((unsigned)T, (unsigned)nh), dim3(AI_WARPS * 32), 0, s, (const TA*)q, q_stride, (const unsigned char*)kc, \
                (const unsigned char*)vc, ksc, vsc, block_table, max_pages, (int)n_pages, token_pos, token_seq, (TA*)out, nh, nkv, d, page_size, span, f, err)
    if (act_dtype == ILLM_BF16) AI_RUN(bf16);
    else if (act_dtype == ILLM_F32) AI_RUN(float);
    else return ILLM_ERR_BAD_ARG;
#undef AI_RUN
    return illm_launch_status();
}
