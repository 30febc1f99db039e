// Element types of the entry points that take more than fp32: sizes, loads and stores of one element or of 16 bytes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

inline bool s2v_dtype_ok(int t)
{
    return t == S2V_F32 || t == S2V_F16 || t == S2V_BF16;
}
inline size_t s2v_dtype_bytes(int t)
{
    return t == S2V_F32 ? 4 : 2;
}

#ifdef __CUDACC__
namespace
{

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
// two fp32 values to one register of two 16-bit ones, the first in the low half
template <typename T> __device__ __forceinline__ uint32_t pack_16bit(float a, float b)
{
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

}  // namespace

// one call of f with a value of the element type that t names
template <typename F>
inline int s2v_by_dtype(int t, F f)
{
    return t == S2V_F32 ? f(float()) : t == S2V_F16 ? f(__half()) : f(__nv_bfloat16());
}
#endif
