// A row's scale and its 8-bit integers, by the definition of s2v_quantize_rows_i8.
#pragma once

#include "elem_types.cuh"

namespace
{

struct q_row {
    float factor, scale;   // factor 0: every integer is 0
    // `largest`: the largest magnitude's bit pattern
    __device__ __forceinline__ explicit q_row(uint32_t largest)
    {
        const float a = __uint_as_float(largest);
        const bool finite = largest < 0x7f800000u, some = finite && a >= 7.703719777548943e-34f;   // 2^-110: below it 127 / a comes near the end of fp32
        factor = some ? __fdiv_rn(127.0f, a) : 0.0f;
        scale = some ? __fdiv_rn(a, 127.0f) : finite ? 0.0f : __uint_as_float(0x7fffffffu);
    }
    // The nearest integer, in the low byte: 1.5 * 2^23 is added, whose last place is one, which rounds the product as rint does and leaves the
    // integer in the low bits (fp32 to integer conversions run at a quarter of the rate of additions).
    __device__ __forceinline__ uint32_t integer(float x) const
    {
        return factor == 0.0f ? 0u : __float_as_uint(__fadd_rn(__fmul_rn(x, factor), 12582912.0f));
    }
    __device__ __forceinline__ uint32_t four(const float* x) const
    {
        return __byte_perm(__byte_perm(integer(x[0]), integer(x[1]), 0x0040), __byte_perm(integer(x[2]), integer(x[3]), 0x0040), 0x5410);
    }
};

// the largest magnitude of a piece of 16 bytes, as the bit pattern of an fp32 number
template <typename T> __device__ __forceinline__ uint32_t q_largest(const uint4& v)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t a = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a = max(a, w[i] & 0x7fffffffu);
        return a;
    } else {   // of both halves at once; 16-bit patterns are in the order of the magnitudes too
#pragma unroll
        for (int i = 0; i < 4; ++i) a = __vmaxu2(a, w[i] & 0x7fff7fffu);
        const uint32_t top = max(a & 0xffffu, a >> 16);
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return top << 16;
        else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)top))) & 0x7fffffffu;
    }
}
// a piece's integers to q
template <typename T> __device__ __forceinline__ void q_store(int8_t* q, bool whole, const uint4& v, const q_row& k)
{
    constexpr int N = PIECE<T>;
    float x[N];
    unpack_piece(v, x, T());
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) w[i] = k.four(x + 4 * i);
    if (whole) {
        if constexpr (N == 4) *reinterpret_cast<uint32_t*>(q) = w[0];
        else *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) q[e] = (int8_t)(w[e / 4] >> (8 * (e & 3)));
    }
}

}  // namespace
