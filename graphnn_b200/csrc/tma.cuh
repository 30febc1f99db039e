// Tensor maps (built on the host, once per call) and the copies that use them.
#pragma once

#include <cuda.h>

#include "common.cuh"

// The driver's encoder, found through the runtime so that the library does not link against the driver.
inline decltype(&cuTensorMapEncodeTiled) s2v_tensor_map_encoder()
{
    static const auto fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(p);
    }();
    return fn;
}

// A [rows x cols] matrix of bytes, rows `ld` bytes apart (a multiple of 16), copied in boxes of `box_rows` rows of 128 bytes in the 128-byte
// swizzle that the matrix instructions read; columns and rows outside the matrix arrive as zeros.
inline bool s2v_byte_matrix_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows)
{
    const auto encode = s2v_tensor_map_encoder();
    if (!encode) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, step[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A row-major output of `es`-byte numbers (S2V_F32, S2V_F16, S2V_BF16), written in boxes of 32 rows of 64 bytes that lie in the 64-byte swizzle.
inline bool s2v_output_map(CUtensorMap* map, int dtype, void* base, int64_t rows, int64_t cols, int64_t ld)
{
    const auto encode = s2v_tensor_map_encoder();
    if (!encode) return false;
    const int es = dtype == S2V_F32 ? 4 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(ld * es)};
    const cuuint32_t box[2] = {(cuuint32_t)(64 / es), 32}, step[2] = {1, 1};
    return encode(map, dtype == S2V_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == S2V_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base,
                  dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

#ifdef __CUDACC__
namespace
{

// the box whose first byte is column `x` (a multiple of 16) of row `y`, to shared memory; arrives on the barrier
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
// the same for a pair of CTAs: the barrier may be the other one's
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y),
                 "r"(bar)
                 : "memory");
}
// a box to the matrix (rows outside are left out; of a row's end every 16 bytes that hold one of its numbers are written, with zeros behind it); x times the
// element size a multiple of 16.  One of the thread's bulk groups.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

}  // namespace
#endif
