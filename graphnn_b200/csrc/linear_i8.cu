// Dense layers with 8-bit weights: rows to 8-bit integers with a scale each, and the entry points of the
// product of two such matrices (gemm_i8.cu).
#include "gemm_i8.cuh"

namespace
{

constexpr float Q_LEAST = 7.703719777548943e-34f;   // 2^-110: below it 127 / a comes near the end of fp32

// A warp per row, two passes over it: the largest magnitude, then the integers.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(int64_t rows, int64_t cols, const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q,
                                                            int64_t ldq, float* __restrict__ scale)
{
    const int lane = threadIdx.x & 31;
    const int64_t warps = ((int64_t)gridDim.x * blockDim.x) >> 5;
    for (int64_t r = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < rows; r += warps) {
        const T* const xr = x + r * ldx;
        int8_t* const qr = q + r * ldq;
        uint32_t a = 0;   // magnitudes as bit patterns: infinities and NaN are the largest
        for (int64_t c = lane; c < cols; c += 32) a = max(a, __float_as_uint(to_f32(xr[c])) & 0x7fffffffu);
        a = __reduce_max_sync(0xffffffffu, a);
        const float amax = __uint_as_float(a);
        const bool finite = a < 0x7f800000u;
        const float f = finite && amax >= Q_LEAST ? __fdiv_rn(127.0f, amax) : 0.0f;
        for (int64_t c = lane; c < cols; c += 32) qr[c] = f == 0.0f ? 0 : (int8_t)__float2int_rn(__fmul_rn(to_f32(xr[c]), f));
        if (lane == 0) scale[r] = !finite ? __uint_as_float(0x7fffffffu) : f == 0.0f ? 0.0f : __fdiv_rn(amax, 127.0f);
    }
}

size_t workspace_scale_offset(int64_t m, int64_t k)
{
    return (size_t)m * (size_t)((k + 15) / 16 * 16);
}

int check_gemm(s2v_ctx* ctx, const char* name, int64_t m, int64_t n, int64_t k, const int8_t* B, int64_t ldb, const float* b_scale, int c_type, const void* C,
               int64_t ldc)
{
    const std::string who(name);
    if (m < 0 || n < 0 || k < 0) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": negative size");
    if (!s2v_dtype_ok(c_type)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": unknown element type");
    if (m == 0 || n == 0) return S2V_OK;
    if (!b_scale || !C || (k > 0 && !B)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": NULL pointer");
    if (k > 131071) return s2v_fail(ctx, S2V_ERR_UNSUPPORTED, who + ": k beyond 131,071, where 32-bit sums can overflow");
    if (m > INT32_MAX || n > INT32_MAX) return s2v_fail(ctx, S2V_ERR_UNSUPPORTED, who + ": more than 2^31 - 1 rows");
    if ((n > 1 && k > 0 && (ldb < k || ldb % 16 != 0)) || (m > 1 && ldc < n))
        return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": leading dimension too small, or of an 8-bit matrix no multiple of 16");
    if (!s2v_aligned16(B)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": 8-bit matrices must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(C) % s2v_dtype_bytes(c_type)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": misaligned output");
    return S2V_OK;
}

}  // namespace

extern "C" {

int s2v_quantize_rows_i8(s2v_ctx* ctx, s2v_stream stream, int64_t rows, int64_t cols, int x_type, const void* x, int64_t ldx, int8_t* q, int64_t ldq,
                         float* scale)
{
    S2V_ENTER(ctx);
    if (rows < 0 || cols < 0) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "quantize_rows: negative size");
    if (!s2v_dtype_ok(x_type)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "quantize_rows: unknown element type");
    if (rows == 0) return S2V_OK;
    if (!scale || (cols > 0 && (!x || !q))) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "quantize_rows: NULL pointer");
    if (rows > 1 && (ldx < cols || ldq < cols)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "quantize_rows: leading dimension below the number of columns");
    if (reinterpret_cast<uintptr_t>(x) % s2v_dtype_bytes(x_type)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "quantize_rows: misaligned x");
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    int64_t blocks = (rows + 7) / 8;
    if (blocks > (int64_t)ctx->sm_count * 8) blocks = (int64_t)ctx->sm_count * 8;
    return s2v_by_dtype(x_type, [&](auto type) {
        using T = decltype(type);
        quantize_rows_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(rows, cols, static_cast<const T*>(x), ldx, q, ldq, scale);
        S2V_CHECK_LAUNCH(ctx, "quantize_rows_kernel");
        return (int)S2V_OK;
    });
}

int s2v_gemm_i8(s2v_ctx* ctx, s2v_stream stream, int64_t m, int64_t n, int64_t k, const int8_t* A, int64_t lda, const float* a_scale, const int8_t* B,
                int64_t ldb, const float* b_scale, const float* bias, int relu, int c_type, void* C, int64_t ldc)
{
    S2V_ENTER(ctx);
    const int rc = check_gemm(ctx, "gemm_i8", m, n, k, B, ldb, b_scale, c_type, C, ldc);
    if (rc != S2V_OK || m == 0 || n == 0) return rc;
    if (!a_scale || (k > 0 && !A)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "gemm_i8: NULL pointer");
    if (m > 1 && k > 0 && (lda < k || lda % 16 != 0)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "gemm_i8: lda below k or no multiple of 16");
    if (!s2v_aligned16(A)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "gemm_i8: 8-bit matrices must be 16-byte aligned");
    const s2v_gemm_i8_args g{m, n, k, lda, ldb, ldc, A, B, a_scale, b_scale, bias, relu, c_type, C};
    return s2v_launch_gemm_i8(ctx, s2v_pick_stream(ctx, stream), g);
}

size_t s2v_linear_i8_workspace_bytes(int64_t m, int64_t k)
{
    if (m <= 0 || k < 0) return 0;
    return workspace_scale_offset(m, k) + (size_t)m * sizeof(float);
}

int s2v_linear_i8(s2v_ctx* ctx, s2v_stream stream, int64_t m, int64_t n, int64_t k, int x_type, const void* x, int64_t ldx, const int8_t* W, int64_t ldw,
                  const float* w_scale, const float* bias, int relu, void* workspace, size_t workspace_bytes, int y_type, void* y, int64_t ldy)
{
    S2V_ENTER(ctx);
    const int rc = check_gemm(ctx, "linear_i8", m, n, k, W, ldw, w_scale, y_type, y, ldy);
    if (rc != S2V_OK || m == 0 || n == 0) return rc;
    if (!s2v_dtype_ok(x_type)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "linear_i8: unknown element type");
    if (!workspace || workspace_bytes < s2v_linear_i8_workspace_bytes(m, k)) return s2v_fail(ctx, S2V_ERR_WORKSPACE, "linear_i8: workspace too small");
    if (!s2v_aligned16(workspace)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "linear_i8: workspace must be 16-byte aligned");
    int8_t* const q = static_cast<int8_t*>(workspace);
    float* const scale = reinterpret_cast<float*>(q + workspace_scale_offset(m, k));
    const int64_t ldq = (k + 15) / 16 * 16;
    const int done = s2v_quantize_rows_i8(ctx, stream, m, k, x_type, x, ldx, q, ldq, scale);
    if (done != S2V_OK) return done;
    return s2v_gemm_i8(ctx, stream, m, n, k, q, ldq, scale, W, ldw, w_scale, bias, relu, y_type, y, ldy);
}

}  // extern "C"
