// What the kernels of adapter products share: the plan as they see it, tensor maps, sizes.
#pragma once
#include "adapters.h"
#include "tc_common.cuh"

struct AdPlan {
    const int *counts, *token_adapter;
    const int4* places;
    const int *groups, *tile_chunk, *chunk_tile, *chunk_groups;
};
static inline AdPlan ad_plan(const int* plan, const AdapterPlanSizes& s) {
    const AdapterPlanLayout l = adapter_plan_layout(s);
    return AdPlan{plan + l.counts, plan + l.token_adapter, (const int4*)(plan + l.places), plan + l.groups, plan + l.tile_chunk, plan + l.chunk_tile, plan + l.chunk_groups};
}

// VEC neighbouring columns
template <int VEC> struct AdColumns;
template <> struct AdColumns<1> {
    __device__ static void load(const float* p, float* f) { f[0] = *p; }
    template <typename T> __device__ static void store(T* p, const float* f) { *p = from_f32<T>(f[0]); }
};
template <> struct AdColumns<4> {
    __device__ static void load(const float* p, float* f) { *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(p); }
    __device__ static void store(float* p, const float* f) { *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(f); }
    __device__ static void store(bf16* p, const float* f) {
        __nv_bfloat162 h[2] = {__floats2bfloat162_rn(f[0], f[1]), __floats2bfloat162_rn(f[2], f[3])};
        *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(h);
    }
};

typedef CUresult (*AdEncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                    const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Tensor map of a row-major bfloat16 matrix [rows, cols]; boxes of [box_rows, box_cols], swizzled over a box's row.
static inline int ad_make_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, int box_rows, int box_cols = TC_BK,
                       CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    static AdEncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
                   ? (AdEncodeTiledFn)p : (AdEncodeTiledFn)nullptr;
    }();
    if (!fn) return ILLM_ERR_BAD_ARG;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)cols * 2};
    cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0 : ILLM_ERR_BAD_ARG;
}

static inline long long ad_round(long long n) { return (n + 255) / 256 * 256; }
static inline int ad_div(long long a, long long b) { return (int)((a + b - 1) / b); }


// adapters_prompt.cu: the prompt form (bfloat16, a plan with tiles)
long long ad_prompt_ws(int T, int N, int K, int chunks);
int ad_prompt_form(const void* x, const void* w, int T, int N, int K, const void* a, const void* b, const float* scales, int count, int R,
                   const AdPlan& plan, int chunks, void* out, int out_dtype, char* ws, int* err, cudaStream_t s);
