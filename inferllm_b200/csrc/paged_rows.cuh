// What the attention kernels over pages of eight-bit or bfloat16 rows share (attention_pages.cu, attention_tiles.cu): copies of scales, reads and
// meetings of a cluster's blocks, and the tensor maps of an entry's pages.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace {

__device__ __forceinline__ void rows_bulk(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// four floats of the same place in another block of the cluster
__device__ __forceinline__ float4 rows_remote4(unsigned at, unsigned rank) {
    unsigned a;
    float4 f;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(a) : "memory");
    return f;
}
__device__ __forceinline__ void rows_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

typedef CUresult (*RowsEncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                      CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// an entry's pages as a matrix [pages * kv heads * page_size, d]; boxes of `box_rows` rows of 128 bytes (eight bits: of d)
int rows_make_map(CUtensorMap* map, const void* ptr, long long rows, int d, int box_rows, bool q8, CUtensorMapSwizzle swizzle) {
    static const RowsEncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) == cudaSuccess && r == cudaDriverEntryPointSuccess ? (RowsEncodeTiledFn)p
                                                                                                                                         : (RowsEncodeTiledFn) nullptr;
    }();
    if (!fn) return ILLM_ERR_BAD_ARG;
    cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)d * (q8 ? 1 : 2)};
    cuuint32_t box[2] = {q8 ? (cuuint32_t)d : 64u, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : ILLM_ERR_BAD_ARG;
}

}  // namespace
