// Tensor maps and the tiled bulk loads that use them (one GPU's own memory, no
// multicast).
#pragma once
#include <cuda.h>

#include "umma.cuh"

namespace ddg {

// 2-D map of `rows` rows of `cols` elements of elem_bytes (1, 4 or 8),
// row_bytes apart; boxes of box_rows x box_cols elements, zeros outside.  base
// and row_bytes are multiples of 16, and so is every box's first column in bytes.
inline int tma_map_2d(CUtensorMap *map, const void *base, int elem_bytes, uint64_t cols, uint64_t rows,
                      uint64_t row_bytes, uint32_t box_cols, uint32_t box_rows)
{
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static thread_local Encode encode = nullptr;  // parties of one process call from threads of their own
    if (!encode) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        DDG_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
        DDG_CHECK(fn && q == cudaDriverEntryPointSuccess, DDG_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
        encode = reinterpret_cast<Encode>(fn);
    }
    const CUtensorMapDataType type = elem_bytes == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : elem_bytes == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32
                                                       : CU_TENSOR_MAP_DATA_TYPE_UINT64;
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {row_bytes};
    const cuuint32_t box[2] = {box_cols, box_rows}, step[2] = {1, 1};
    const CUresult r = encode(map, type, 2, const_cast<void *>(base), dims, strides, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    DDG_CHECK(r == CUDA_SUCCESS, DDG_ERR_CUDA, "tensor map of %llu x %llu elements refused (driver error %d)",
              (unsigned long long)rows, (unsigned long long)cols, int(r));
    return DDG_OK;
}

__device__ __forceinline__ void tma_prefetch(const CUtensorMap *map)
{
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, int col, int row, uint64_t *bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(col), "r"(row), "r"(smem_addr(bar))
        : "memory");
}

}  // namespace ddg
