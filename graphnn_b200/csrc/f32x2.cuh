// Two fp32 numbers in one 64-bit register: additions, products and multiply-adds of both by one instruction, each rounded as the single ones are (but for a product that an addition follows: the two may
// be made one multiply-add).
#pragma once

#include "elem_types.cuh"

namespace
{

__device__ __forceinline__ uint64_t f2_of(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 f2_get(uint64_t v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float f2_sum(uint64_t v)
{
    const float2 f = f2_get(v);
    return f.x + f.y;
}

// a piece of 16 bytes as pairs
template <typename T> __device__ __forceinline__ void f2_unpack(const uint4& v, uint64_t* x)
{
    float f[PIECE<T>];
    unpack_piece(v, f, T());
#pragma unroll
    for (int i = 0; i < PIECE<T> / 2; ++i) x[i] = f2_of(f[2 * i], f[2 * i + 1]);
}
template <typename T> __device__ __forceinline__ uint4 f2_piece(const uint64_t* x)
{
    float f[PIECE<T>];
#pragma unroll
    for (int i = 0; i < PIECE<T> / 2; ++i) {
        const float2 p = f2_get(x[i]);
        f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
    return pack_piece(f, T());
}
// Four 8-bit integers of a word as two pairs: each byte, with its sign turned, is put under the exponent of 2^23, where a unit is the last place, and 2^23 + 128
// taken away, exactly (conversions run at a quarter of the rate).
__device__ __forceinline__ void f2_unpack8(uint32_t w, uint64_t* x)
{
    const uint64_t away = f2_of(-8388736.0f, -8388736.0f);
    w ^= 0x80808080u;
    x[0] = f2_add(f2_of(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441))), away);
    x[1] = f2_add(f2_of(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443))), away);
}

}  // namespace
