// The weight gradient of a dense layer whose input was kept as 8-bit rows:  dW = dy^T (scale q),  dbias = sum of dy over the rows.
#include "product_simt.cuh"

namespace
{

struct scaled_i8_across_k {   // element (column, row) of scale[row] * q[row][column]
    static constexpr bool K_FAST = false;
    const int8_t* q;
    int64_t ld;
    const float* scale;
    __device__ __forceinline__ float operator()(int64_t i, int64_t k) const { return (float)q[k * ld + i] * scale[k]; }
};

// sums of columns: 32 columns a CTA, 8 threads each, the rows in turn
template <typename T> __global__ void __launch_bounds__(256) column_sums_kernel(int64_t rows, int64_t cols, const T* __restrict__ x, int64_t ldx, float* __restrict__ out)
{
    __shared__ float part[8][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int g = threadIdx.x >> 5;
    float t = 0.0f;
    if (c < cols)
        for (int64_t r = g; r < rows; r += 8) t += to_f32(x[r * ldx + c]);
    part[g][threadIdx.x & 31] = t;
    __syncthreads();
    if (g || c >= cols) return;
    t = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += part[i][threadIdx.x & 31];
    out[c] = t;
}

}  // namespace

extern "C" {

size_t s2v_linear_i8_grad_workspace_bytes(int64_t m, int64_t n, int64_t k, int dy_type)
{
    if (m <= 0 || n <= 0 || k <= 0 || !s2v_dtype_ok(dy_type)) return 0;
    return 256;
}

int s2v_linear_i8_grad(s2v_ctx* ctx, s2v_stream stream, int64_t m, int64_t n, int64_t k, int dy_type, const void* dy, int64_t lddy, const int8_t* q, int64_t ldq,
                       const float* q_scale, void* workspace, size_t workspace_bytes, void* dW, int64_t lddw, float* dbias)
{
    S2V_ENTER(ctx);
    const auto bad = [&](int status, const char* what) { return s2v_fail(ctx, status, std::string("linear_i8_grad: ") + what); };
    if (m < 0 || n < 0 || k < 0) return bad(S2V_ERR_INVALID_ARG, "negative size");
    if (!s2v_dtype_ok(dy_type)) return bad(S2V_ERR_INVALID_ARG, "unknown element type");
    if (n == 0) return S2V_OK;
    if (m > INT32_MAX || n > INT32_MAX || k > INT32_MAX) return bad(S2V_ERR_UNSUPPORTED, "a size above 2^31 - 1");
    const int64_t es = (int64_t)s2v_dtype_bytes(dy_type);
    if ((k > 0 && !dW) || (m > 0 && (!dy || (k > 0 && (!q || !q_scale))))) return bad(S2V_ERR_INVALID_ARG, "NULL pointer");
    if ((m > 1 && (lddy < n || (k > 0 && ldq < k))) || (n > 1 && lddw < k)) return bad(S2V_ERR_INVALID_ARG, "leading dimension below the number of columns");
    if (reinterpret_cast<uintptr_t>(dy) % es || reinterpret_cast<uintptr_t>(dW) % es || !s2v_aligned4(q_scale, dbias)) return bad(S2V_ERR_INVALID_ARG, "misaligned pointer");
    if (workspace_bytes < s2v_linear_i8_grad_workspace_bytes(m, n, k, dy_type) || (!workspace && workspace_bytes)) return bad(S2V_ERR_WORKSPACE, "workspace too small");
    if (!s2v_aligned16(workspace)) return bad(S2V_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    return s2v_by_dtype(dy_type, [&](auto type) {
        using T = decltype(type);
        if (dbias) {
            column_sums_kernel<T><<<(unsigned)((n + 31) / 32), 256, 0, st>>>(m, n, static_cast<const T*>(dy), lddy, dbias);
            S2V_CHECK_LAUNCH(ctx, "column_sums_kernel");
        }
        return product_simt(ctx, st, "linear_i8_grad", n, k, m, across_k<T>{static_cast<const T*>(dy), lddy}, scaled_i8_across_k{q, ldq, q_scale},
                            store_outputs<T>{static_cast<T*>(dW), lddw, n, k});
    });
}

}  // extern "C"
