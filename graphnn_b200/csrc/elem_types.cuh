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
// whether arrays of 32-bit numbers (NULL ones among them) lie as a kernel's loads and stores need them
template <typename... P> inline bool s2v_aligned4(const P*... p)
{
    return ((reinterpret_cast<uintptr_t>(p) | ...) & 3u) == 0;
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
// ---- pieces of 16 bytes
template <typename T> constexpr int PIECE = 16 / (int)sizeof(T);   // elements of one

__device__ __forceinline__ void unpack_piece(const uint4& v, float* x, float)
{
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack_piece(const uint4& v, float* x, __half)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack_piece(const uint4& v, float* x, __nv_bfloat16)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ uint4 pack_piece(const float* y, float) { return make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])); }
template <typename T> __device__ __forceinline__ uint4 pack_piece(const float* y, T)
{
    return make_uint4(pack_16bit<T>(y[0], y[1]), pack_16bit<T>(y[2], y[3]), pack_16bit<T>(y[4], y[5]), pack_16bit<T>(y[6], y[7]));
}

// A row's columns: `head` in front of the first 16-byte boundary, `pieces` of 16 bytes, `tail` behind them.
template <typename T> struct row_pieces {
    int head, tail;
    int pieces;
    __device__ __forceinline__ row_pieces(const T* z, int64_t cols)
    {
        const int off = (int)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / (int)sizeof(T);
        head = off < cols ? off : (int)cols;
        pieces = (int)((cols - head) / PIECE<T>);
        tail = (int)(cols - head - (int64_t)pieces * PIECE<T>);
    }
};

}  // namespace

// one call of f with a value of the element type that t names
template <typename F>
inline int s2v_by_dtype(int t, F f)
{
    return t == S2V_F32 ? f(float()) : t == S2V_F16 ? f(__half()) : f(__nv_bfloat16());
}
#endif
