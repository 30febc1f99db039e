// A product of any two matrices in fp32 arithmetic, 64 x 64 outputs a CTA: where the operands lie and what becomes of the outputs is the caller's.
#pragma once

#include "elem_types.cuh"

namespace
{

// element (i, k) of an operand whose rows lie along k, or across it
template <typename T> struct along_k {
    static constexpr bool K_FAST = true;
    const T* p;
    int64_t ld;
    __device__ __forceinline__ float operator()(int64_t i, int64_t k) const { return to_f32(p[i * ld + k]); }
};
template <typename T> struct across_k {
    static constexpr bool K_FAST = false;
    const T* p;
    int64_t ld;
    __device__ __forceinline__ float operator()(int64_t i, int64_t k) const { return to_f32(p[k * ld + i]); }
};

constexpr int PS_TILE = 64, PS_K = 16, PS_THREADS = 256;

// out(row, column, four rows by four columns of this thread: 4 * (thread / 16) and 4 * (thread % 16) of the tile)
template <class A, class B, class OUT> __global__ void __launch_bounds__(PS_THREADS) product_simt_kernel(int64_t m, int64_t n, int64_t k, int n_tiles, A a, B b, OUT out)
{
    __shared__ float as[PS_K][PS_TILE + 4], bs[PS_K][PS_TILE + 4];
    const int64_t row0 = (int64_t)(blockIdx.x / n_tiles) * PS_TILE, col0 = (int64_t)(blockIdx.x % n_tiles) * PS_TILE;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < k; k0 += PS_K) {
#pragma unroll
        for (int u = 0; u < PS_TILE * PS_K / PS_THREADS; ++u) {
            const int at = threadIdx.x + u * PS_THREADS;
            const int ak = A::K_FAST ? at % PS_K : at / PS_TILE, ai = A::K_FAST ? at / PS_K : at % PS_TILE;
            const int bk = B::K_FAST ? at % PS_K : at / PS_TILE, bi = B::K_FAST ? at / PS_K : at % PS_TILE;
            as[ak][ai] = row0 + ai < m && k0 + ak < k ? a(row0 + ai, k0 + ak) : 0.0f;
            bs[bk][bi] = col0 + bi < n && k0 + bk < k ? b(col0 + bi, k0 + bk) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PS_K; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(&as[i][4 * ty]), y = *reinterpret_cast<const float4*>(&bs[i][4 * tx]);
            const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[r][c] = fmaf(xs[r], ys[c], acc[r][c]);
        }
        __syncthreads();
    }
    out(row0 + 4 * ty, col0 + 4 * tx, acc);
}

template <class A, class B, class OUT> int product_simt(s2v_ctx* ctx, cudaStream_t st, const char* name, int64_t m, int64_t n, int64_t k, A a, B b, OUT out)
{
    const int64_t mt = (m + PS_TILE - 1) / PS_TILE, nt = (n + PS_TILE - 1) / PS_TILE;
    if (mt == 0 || nt == 0) return S2V_OK;
    if (nt > INT32_MAX || mt > INT32_MAX / nt) return s2v_fail(ctx, S2V_ERR_UNSUPPORTED, std::string(name) + ": more than 2^31 tiles of outputs");
    product_simt_kernel<<<(unsigned)(mt * nt), PS_THREADS, 0, st>>>(m, n, k, (int)nt, a, b, out);
    S2V_CHECK_LAUNCH(ctx, name);
    return S2V_OK;
}

// the outputs as they are
template <typename T> struct store_outputs {
    T* p;
    int64_t ld, m, n;
    __device__ __forceinline__ void operator()(int64_t r0, int64_t c0, const float (&acc)[4][4]) const
    {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (r0 + r < m && c0 + c < n) p[(r0 + r) * ld + c0 + c] = from_f32<T>(acc[r][c]);
    }
};

}  // namespace
