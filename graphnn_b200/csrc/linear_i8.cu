// Dense layers with 8-bit weights: rows to 8-bit integers with a scale each, and the entry points of the
// product of two such matrices (gemm_i8.cu).
#include "gemm_i8.cuh"
#include "quantize.cuh"

namespace
{

constexpr int QR_CTA = 256;

// A row by a warp (THREADS = 32) or by a CTA: 16-byte pieces, the first NV of each thread kept in registers between the largest magnitude and the
// integers (a longer row's others are read again), the last reads of x marked as such, so that L2 keeps the integers for a product behind this kernel
// (491,520 x 128 fp32 and the product with 256 channels: 152 us, else 156); single columns in front of the first 16-byte boundary and behind the last piece.
template <typename T, int NV, int THREADS>
__global__ void __launch_bounds__(QR_CTA) quantize_rows_kernel(int64_t rows, int64_t cols, const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q,
                                                               int64_t ldq, float* __restrict__ scale)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (a product behind this kernel waits for its end by itself)
    constexpr int N = PIECE<T>;
    __shared__ uint32_t part[QR_CTA / 32];
    const int at = THREADS == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t own = THREADS == 32 ? (int64_t)blockIdx.x * (QR_CTA / 32) + (threadIdx.x >> 5) : blockIdx.x, step = (int64_t)gridDim.x * (QR_CTA / THREADS);
    for (int64_t r = own; r < rows; r += step) {
        const T* const xr = x + r * ldx;
        int8_t* const qr = q + r * ldq;
        const row_pieces<T> row(xr, cols);
        const uint4* const xp = reinterpret_cast<const uint4*>(xr + row.head);
        uint4 v[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < row.pieces) v[j] = __ldcs(xp + j * THREADS + at);
        const bool single = at < row.head || (at >= THREADS - row.tail);
        const int64_t single_at = at < row.head ? at : cols - THREADS + at;
        const float xs = single ? to_f32(xr[single_at]) : 0.0f;
        uint32_t a = __float_as_uint(xs) & 0x7fffffffu;   // magnitudes as bit patterns: infinities and NaN are the largest
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < row.pieces) a = max(a, q_largest<T>(v[j]));
        for (int64_t p = NV * THREADS + at; p < row.pieces; p += THREADS) a = max(a, q_largest<T>(__ldg(xp + p)));
        a = __reduce_max_sync(0xffffffffu, a);
        if constexpr (THREADS > 32) {
            __syncthreads();   // (the row before has been read)
            if ((at & 31) == 0) part[at >> 5] = a;
            __syncthreads();
            a = __reduce_max_sync(0xffffffffu, part[at & (QR_CTA / 32 - 1)]);
        }
        const q_row k(a);
        int8_t* const qp = qr + row.head;
        const bool whole = (reinterpret_cast<uintptr_t>(qp) & (N - 1)) == 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < row.pieces) q_store<T>(qp + (j * THREADS + at) * N, whole, v[j], k);
        for (int64_t p = NV * THREADS + at; p < row.pieces; p += THREADS) q_store<T>(qp + p * N, whole, __ldcs(xp + p), k);
        if (single) qr[single_at] = (int8_t)k.integer(xs);
        if (at == 0) scale[r] = k.scale;
    }
}

// Short rows: LANES lanes a row with NV pieces each, so that what a row needs once (its place, the reduction, the divisions) is done for 32 / LANES
// rows by the same instructions.
template <typename T, int LANES, int NV>
__global__ void __launch_bounds__(QR_CTA) quantize_short_rows_kernel(int64_t rows, int64_t cols, const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q,
                                                                     int64_t ldq, float* __restrict__ scale)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (a product behind this kernel waits for its end by itself)
    constexpr int N = PIECE<T>, GROUPS = QR_CTA / LANES;
    static_assert(LANES >= N - 1, "the columns of the head, or of the tail, have a lane each");
    const int at = threadIdx.x % LANES;
    for (int64_t first = (int64_t)blockIdx.x * GROUPS; first < rows; first += (int64_t)gridDim.x * GROUPS) {
        const int64_t r = min(first + threadIdx.x / LANES, rows - 1);   // (the last row, several times over, where there are no more)
        const T* const xr = x + r * ldx;
        int8_t* const qr = q + r * ldq;
        const row_pieces<T> row(xr, cols);
        const uint4* const xp = reinterpret_cast<const uint4*>(xr + row.head) + at;
        uint4 v[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = j * LANES + at < row.pieces ? __ldcs(xp + j * LANES) : make_uint4(0, 0, 0, 0);
        const float x0 = at < row.head ? to_f32(xr[at]) : 0.0f, x1 = at < row.tail ? to_f32(xr[cols - row.tail + at]) : 0.0f;
        uint32_t a = max(__float_as_uint(x0) & 0x7fffffffu, __float_as_uint(x1) & 0x7fffffffu);   // the largest magnitude's bit pattern
#pragma unroll
        for (int j = 0; j < NV; ++j) a = max(a, q_largest<T>(v[j]));
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
        const q_row k(a);
        int8_t* const qp = qr + row.head;
        const bool whole = (reinterpret_cast<uintptr_t>(qp) & (N - 1)) == 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * LANES + at < row.pieces) q_store<T>(qp + (j * LANES + at) * N, whole, v[j], k);
        if (at < row.head) qr[at] = (int8_t)k.integer(x0);
        if (at < row.tail) qr[cols - row.tail + at] = (int8_t)k.integer(x1);
        if (at == 0) scale[r] = k.scale;
    }
}

template <typename T> int quantize_launch(s2v_ctx* ctx, cudaStream_t st, int64_t rows, int64_t cols, const T* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale)
{
    const int64_t pieces = cols / PIECE<T>;
    const auto go = [&](auto kernel, int64_t per_block) {
        const int64_t blocks = (rows + per_block - 1) / per_block, cap = (int64_t)1 << 20;
        kernel<<<(unsigned)(blocks < cap ? blocks : cap), QR_CTA, 0, st>>>(rows, cols, x, ldx, q, ldq, scale);
        S2V_CHECK_LAUNCH(ctx, "quantize_rows_kernel");
        return (int)S2V_OK;
    };
    if (pieces <= 8) return go(quantize_short_rows_kernel<T, 8, 1>, QR_CTA / 8);
    if (pieces <= 32) return go(quantize_short_rows_kernel<T, 8, 4>, QR_CTA / 8);
    if (pieces <= 64) return go(quantize_short_rows_kernel<T, 8, 8>, QR_CTA / 8);
    if (pieces <= 128) return go(quantize_rows_kernel<T, 4, 32>, QR_CTA / 32);
    if (pieces <= 2 * QR_CTA) return go(quantize_rows_kernel<T, 2, QR_CTA>, 1);
    if (pieces <= 4 * QR_CTA) return go(quantize_rows_kernel<T, 4, QR_CTA>, 1);
    return go(quantize_rows_kernel<T, 8, QR_CTA>, 1);
}

int check_quantize(s2v_ctx* ctx, const char* name, int64_t rows, int64_t cols, int x_type, const void* x, int64_t ldx)
{
    const auto bad = [&](int status, const char* what) { return s2v_fail(ctx, status, std::string(name) + ": " + what); };
    if (rows < 0 || cols < 0) return bad(S2V_ERR_INVALID_ARG, "negative size");
    if (!s2v_dtype_ok(x_type)) return bad(S2V_ERR_INVALID_ARG, "unknown element type");
    if (rows == 0) return S2V_OK;
    if (cols > INT32_MAX) return bad(S2V_ERR_UNSUPPORTED, "more than 2^31 - 1 columns");
    if (cols > 0 && !x) return bad(S2V_ERR_INVALID_ARG, "NULL pointer");
    if (rows > 1 && ldx < cols) return bad(S2V_ERR_INVALID_ARG, "leading dimension below the number of columns");
    if (reinterpret_cast<uintptr_t>(x) % s2v_dtype_bytes(x_type)) return bad(S2V_ERR_INVALID_ARG, "misaligned x");
    return S2V_OK;
}

size_t workspace_scale_offset(int64_t m, int64_t k)
{
    return (size_t)m * (size_t)((k + 15) / 16 * 16);
}

int check_gemm(s2v_ctx* ctx, const char* name, int64_t m, int64_t n, int64_t k, const int8_t* B, int64_t ldb, const float* b_scale, const float* bias, int c_type,
               const void* C, int64_t ldc)
{
    const auto bad = [&](int status, const char* what) { return s2v_fail(ctx, status, std::string(name) + ": " + what); };
    if (m < 0 || n < 0 || k < 0) return bad(S2V_ERR_INVALID_ARG, "negative size");
    if (!s2v_dtype_ok(c_type)) return bad(S2V_ERR_INVALID_ARG, "unknown element type");
    if (m == 0 || n == 0) return S2V_OK;
    if (!b_scale || !C || (k > 0 && !B)) return bad(S2V_ERR_INVALID_ARG, "NULL pointer");
    if (k > 131071) return bad(S2V_ERR_UNSUPPORTED, "k beyond 131,071, where 32-bit sums can overflow");
    if (m > INT32_MAX || n > INT32_MAX) return bad(S2V_ERR_UNSUPPORTED, "more than 2^31 - 1 rows");
    if ((n > 1 && k > 0 && (ldb < k || ldb % 16 != 0)) || (m > 1 && ldc < n))
        return bad(S2V_ERR_INVALID_ARG, "leading dimension too small, or of an 8-bit matrix no multiple of 16");
    if (!s2v_aligned16(B)) return bad(S2V_ERR_INVALID_ARG, "8-bit matrices must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(C) % s2v_dtype_bytes(c_type)) return bad(S2V_ERR_INVALID_ARG, "misaligned output");
    if (!s2v_aligned4(b_scale, bias)) return bad(S2V_ERR_INVALID_ARG, "misaligned scales or bias");
    return S2V_OK;
}

}  // namespace

extern "C" {

int s2v_quantize_rows_i8(s2v_ctx* ctx, s2v_stream stream, int64_t rows, int64_t cols, int x_type, const void* x, int64_t ldx, int8_t* q, int64_t ldq,
                         float* scale)
{
    S2V_ENTER(ctx);
    const int rc = check_quantize(ctx, "quantize_rows", rows, cols, x_type, x, ldx);
    if (rc != S2V_OK || rows == 0) return rc;
    if (!scale || (cols > 0 && !q)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "quantize_rows: NULL pointer");
    if (!s2v_aligned4(scale)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "quantize_rows: misaligned scale");
    if (rows > 1 && ldq < cols) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "quantize_rows: leading dimension below the number of columns");
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    return s2v_by_dtype(x_type, [&](auto type) {
        using T = decltype(type);
        return quantize_launch<T>(ctx, st, rows, cols, static_cast<const T*>(x), ldx, q, ldq, scale);
    });
}

int s2v_gemm_i8(s2v_ctx* ctx, s2v_stream stream, int64_t m, int64_t n, int64_t k, const int8_t* A, int64_t lda, const float* a_scale, const int8_t* B,
                int64_t ldb, const float* b_scale, const float* bias, int relu, int c_type, void* C, int64_t ldc)
{
    S2V_ENTER(ctx);
    const int rc = check_gemm(ctx, "gemm_i8", m, n, k, B, ldb, b_scale, bias, c_type, C, ldc);
    if (rc != S2V_OK || m == 0 || n == 0) return rc;
    if (!a_scale || (k > 0 && !A)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "gemm_i8: NULL pointer");
    if (m > 1 && k > 0 && (lda < k || lda % 16 != 0)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "gemm_i8: lda below k or no multiple of 16");
    if (!s2v_aligned16(A)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "gemm_i8: 8-bit matrices must be 16-byte aligned");
    if (!s2v_aligned4(a_scale)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "gemm_i8: misaligned scales");
    const s2v_gemm_i8_args g{m, n, k, lda, ldb, ldc, A, B, a_scale, b_scale, bias, relu, c_type, C};
    return s2v_launch_gemm_i8(ctx, s2v_pick_stream(ctx, stream), g, false);
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
    const int rc = check_gemm(ctx, "linear_i8", m, n, k, W, ldw, w_scale, bias, y_type, y, ldy);
    if (rc != S2V_OK || m == 0 || n == 0) return rc;
    if (!s2v_dtype_ok(x_type)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "linear_i8: unknown element type");
    if (!workspace || workspace_bytes < s2v_linear_i8_workspace_bytes(m, k)) return s2v_fail(ctx, S2V_ERR_WORKSPACE, "linear_i8: workspace too small");
    if (!s2v_aligned16(workspace)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "linear_i8: workspace must be 16-byte aligned");
    int8_t* const q = static_cast<int8_t*>(workspace);
    float* const scale = reinterpret_cast<float*>(q + workspace_scale_offset(m, k));
    const int64_t ldq = (k + 15) / 16 * 16;
    const int bad = check_quantize(ctx, "linear_i8", m, k, x_type, x, ldx);
    if (bad != S2V_OK) return bad;
    s2v_gemm_i8_args g{m, n, k, ldx, ldw, ldy, x, W, nullptr, w_scale, bias, relu, y_type, y};
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    if (s2v_gemv_i8_takes(m, n, k)) return s2v_launch_gemv_i8(ctx, st, x_type, g);
    const int quantized = s2v_by_dtype(x_type, [&](auto type) { return quantize_launch<decltype(type)>(ctx, st, m, k, static_cast<const decltype(type)*>(x), ldx, q, ldq, scale); });
    if (quantized != S2V_OK) return quantized;
    g.lda = ldq, g.A = q, g.a_scale = scale;
    return s2v_launch_gemm_i8(ctx, st, g, true);
}

}  // extern "C"
