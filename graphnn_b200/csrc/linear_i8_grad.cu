// The weight gradient of a dense layer whose input was kept as 8-bit rows:  dW = dy^T (scale q),  dbias = sum of dy over the rows.
//
// The rows' scales go to dy, in fp32:  dW_jl = sum_i (dy_ij scale_i) q_il.  8-bit integers are exact in 16 bits, so one rounding is left, that of dy_ij scale_i to
// the 16 bits that the tensor cores multiply: half a step of bf16 or fp16, as dy itself has; fp32 goes as three bf16 numbers.  For fp16 a column is
// first scaled by a power of two that puts its largest product's binade at 2^14, since scale_i can take dy_ij out of fp16's normal range; dW's row is scaled back.
// Where dW is small and the rows are many, that and the products are one kernel (linear_i8_direct.cu); else both matrices are written in 16 bits first, which many
// tiles then read.
#include <algorithm>

#include "linear_i8_grad.cuh"

namespace
{

constexpr int LG_THREADS = 256;
constexpr int LG_SLABS = 592;   // shares of the rows at most (four CTAs on each of 148 SMs)

struct LgRows {
    int64_t m, n, lddy, share;   // rows of a CTA
    const void* dy;
    const float* scale;
    const float* factor;         // of columns, fp16 alone
    int wide, groups;            // groups: of eight columns in a CTA, a power of two up to 32
    uint16_t* out;
    int64_t ldo, part;
    float* lines;                // [slabs][n]
};

// Eight columns a thread, the rows of a share in turn: PACK: their products with the scales in 16 bits, and the sums of dy; else the largest finite products.
template <typename T, bool PACK> __global__ void __launch_bounds__(LG_THREADS) grad_rows_kernel(const LgRows a)
{
    __shared__ float of[8][LG_THREADS + 1];
    const int group = threadIdx.x % a.groups, lane = threadIdx.x / a.groups, lanes = LG_THREADS / a.groups;
    const int64_t col = ((int64_t)blockIdx.x * a.groups + group) * 8, from = blockIdx.y * a.share, to = min(a.m, from + a.share);
    const int cols = (int)max((int64_t)0, min((int64_t)8, a.n - col));
    float t[8] = {}, factor[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) factor[e] = PACK && a.factor && e < cols ? a.factor[col + e] : 1.0f;
    if (cols > 0)
        for (int64_t r = from + lane; r < to; r += lanes) {
            const T* const p = static_cast<const T*>(a.dy) + r * a.lddy + col;
            const float s = a.scale[r];
            float f[8];
            if (a.wide && cols == 8) {
#pragma unroll
                for (int c = 0; c < 8; c += PIECE<T>) unpack_piece(*reinterpret_cast<const uint4*>(p + c), f + c, T());
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = e < cols ? to_f32(p[e]) : 0.0f;
            }
            if constexpr (PACK) {
                uint16_t* const to16 = a.out + r * a.ldo + col;
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] += f[e], f[e] = f[e] * s * factor[e];
                constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
                using H = typename std::conditional<std::is_same<T, __half>::value, __half, __nv_bfloat16>::type;
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        h[j] = PARTS > 1 ? mm16_head(f[2 * j], f[2 * j + 1]) : pack_16bit<H>(f[2 * j], f[2 * j + 1]);
                        if (PARTS > 1) f[2 * j] -= __uint_as_float(h[j] << 16), f[2 * j + 1] -= __uint_as_float(h[j] & 0xffff0000u);
                    }
                    *reinterpret_cast<uint4*>(to16 + q * a.part) = make_uint4(h[0], h[1], h[2], h[3]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = fabsf(f[e] * s);
                    if (v < INFINITY) t[e] = fmaxf(t[e], v);
                }
            }
        }
#pragma unroll
    for (int e = 0; e < 8; ++e) of[e][threadIdx.x] = t[e];
    __syncthreads();
    for (int i = threadIdx.x; i < a.groups * 8; i += LG_THREADS) {
        const int g = i / 8, e = i % 8;
        const int64_t c = ((int64_t)blockIdx.x * a.groups + g) * 8 + e;
        if (c >= a.n) continue;
        float v = 0.0f;
        for (int l = 0; l < lanes; ++l) v = PACK ? v + of[e][l * a.groups + g] : fmaxf(v, of[e][l * a.groups + g]);
        a.lines[blockIdx.y * a.n + c] = v;
    }
}
// Lines of sums to dbias, or of largest products to the columns' factors (factor[n], then their inverses).
template <bool SUMS> __global__ void __launch_bounds__(256) grad_lines_kernel(int lines, int64_t n, const float* __restrict__ from, float* __restrict__ out)
{
    __shared__ float part[8][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int g = threadIdx.x >> 5;
    float t = 0.0f;
    if (c < n)
        for (int l = g; l < lines; l += 8) t = SUMS ? t + from[l * n + c] : fmaxf(t, from[l * n + c]);
    part[g][threadIdx.x & 31] = t;
    __syncthreads();
    if (g || c >= n) return;
    t = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t = SUMS ? t + part[i][threadIdx.x & 31] : fmaxf(t, part[i][threadIdx.x & 31]);
    if (SUMS) out[c] = t;
    else {
        const int e = min(max((int)(__float_as_uint(t) >> 23) - 127, -100), 127);   // (products below 2^-100 are not scaled up further)
        out[c] = exp2f((float)(14 - e)), out[n + c] = exp2f((float)(e - 14));
    }
}
// 8-bit integers as 16-bit numbers, eight a thread
template <typename H> __global__ void __launch_bounds__(256) grad_q_kernel(int64_t rows, int64_t cols, const int8_t* __restrict__ q, int64_t ldq, int wide, uint16_t* __restrict__ out, int64_t ldo)
{
    const int64_t per_row = (cols + 7) / 8, all = rows * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row, col = (i - row * per_row) * 8;
        const int8_t* const from = q + row * ldq + col;
        int8_t b[8];
        if (wide && col + 8 <= cols) *reinterpret_cast<uint2*>(b) = *reinterpret_cast<const uint2*>(from);
        else {
#pragma unroll
            for (int e = 0; e < 8; ++e) b[e] = col + e < cols ? from[e] : (int8_t)0;
        }
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = pack_16bit<H>((float)b[2 * j], (float)b[2 * j + 1]);
        *reinterpret_cast<uint4*>(out + row * ldo + col) = make_uint4(h[0], h[1], h[2], h[3]);
    }
}

// Few rows: fp32 arithmetic and one launch.  64 rows of dW by 256 columns a CTA, 8 x 8 a thread with its columns 32 apart, so that reads of q and writes of dW are a
// warp's neighbours wherever rows lie.
constexpr int LG_FEW = 32;   // rows
// ... and up to so many multiply-adds: a call of 4 x 177 x 137 fp32 takes 19 us, 25 by the other forms' four launches or five; of 32 x 4096 x 4096 bf16 (2^29) 60 and 32
constexpr int64_t LG_FEW_PRODUCTS = (int64_t)1 << 26;
template <typename T>
__global__ void __launch_bounds__(256) grad_few_kernel(int m, int64_t n, int64_t k, const T* __restrict__ dy, int64_t lddy, const int8_t* __restrict__ q, int64_t ldq, const float* __restrict__ scale,
                                                       T* __restrict__ dW, int64_t lddw, float* __restrict__ dbias)
{
    __shared__ __align__(16) float of[LG_FEW][64];   // dy times the rows' scales
    const int64_t row0 = (int64_t)blockIdx.y * 64, col0 = (int64_t)blockIdx.x * 256 + (threadIdx.x & 31);
    for (int i = threadIdx.x; i < m * 64; i += 256) {
        const int64_t j = row0 + (i & 63);
        of[i >> 6][i & 63] = j < n ? to_f32(dy[(i >> 6) * lddy + j]) * scale[i >> 6] : 0.0f;
    }
    if (dbias && blockIdx.x == 0 && threadIdx.x < 64 && row0 + threadIdx.x < n) {
        float t = 0.0f;
        for (int i = 0; i < m; ++i) t += to_f32(dy[i * lddy + row0 + threadIdx.x]);
        dbias[row0 + threadIdx.x] = t;
    }
    __syncthreads();
    const int r0 = (threadIdx.x >> 5) * 8;
    float acc[8][8] = {};
#pragma unroll 2
    for (int i = 0; i < m; ++i) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = col0 + 32 * e < k ? (float)q[i * ldq + col0 + 32 * e] : 0.0f;
        const float4 a = *reinterpret_cast<const float4*>(&of[i][r0]), b = *reinterpret_cast<const float4*>(&of[i][r0 + 4]);
        const float y[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[r][e] = fmaf(y[r], x[e], acc[r][e]);
    }
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (row0 + r0 + r < n && col0 + 32 * e < k) dW[(row0 + r0 + r) * lddw + col0 + 32 * e] = from_f32<T>(acc[r][e]);
}

// Where things lie in the workspace.  Matrices in 16 bits are made for a piece of the rows at a time, dW's sums of several pieces kept in fp32.
constexpr size_t LG_BYTES = (size_t)256 << 20;   // of a piece, about
struct LgSpace {
    size_t dy = 0, q = 0, columns = 0, factor = 0, lines = 0, sum = 0, bytes = 0;
    int64_t ldn = 0, ldk = 0, parts = 0, piece = 0, pieces = 1, slabs = LG_SLABS;   // slabs: of a piece
    LgSpace(int64_t m, int64_t n, int64_t k, int type, bool direct)
    {
        const auto take = [&](size_t& at, size_t size) { at = bytes, bytes += (size + 255) / 256 * 256; };
        parts = type == S2V_F32 ? 3 : 1;
        ldn = (n + 7) / 8 * 8, ldk = (k + 7) / 8 * 8;
        if (!direct) {
            piece = std::min(m, std::max<int64_t>(4096, (int64_t)(LG_BYTES / (size_t)(ldn * 2 * parts + ldk * 2)) / 64 * 64)), pieces = (m + piece - 1) / piece;
            slabs = std::max<int64_t>(1, LG_SLABS / pieces);
            take(dy, (size_t)piece * ldn * 2 * parts), take(q, (size_t)piece * ldk * 2);
            if (pieces > 1) take(sum, (size_t)n * mm16_pitch(k) * sizeof(float));
        }
        take(columns, (size_t)std::max<int64_t>(pieces * slabs, LG_SLABS) * n * sizeof(float));
        take(factor, (size_t)n * 2 * sizeof(float));
        take(lines, direct ? linear_i8_direct_floats(m, n, k) * sizeof(float) : mm16_lines_bytes(piece, (int)parts));
    }
};

}  // namespace

extern "C" {

size_t s2v_linear_i8_grad_workspace_bytes(int64_t m, int64_t n, int64_t k, int dy_type)
{
    if (m <= 0 || n <= 0 || k <= 0 || m > INT32_MAX || n > INT32_MAX || k > INT32_MAX || !s2v_dtype_ok(dy_type)) return 0;
    if (!mm16_size_ok(m, n) || !mm16_size_ok(m, k) || !mm16_size_ok(n, k)) return 0;
    // (rows that don't lie on 16-byte boundaries take the other way)
    return std::max(LgSpace(m, n, k, dy_type, false).bytes, linear_i8_direct_takes(m, n, k, dy_type) ? LgSpace(m, n, k, dy_type, true).bytes : 0) + MM16_SLACK;
}

int s2v_linear_i8_grad(s2v_ctx* ctx, s2v_stream stream, int64_t m, int64_t n, int64_t k, int dy_type, const void* dy, int64_t lddy, const int8_t* q, int64_t ldq,
                       const float* q_scale, void* workspace, size_t workspace_bytes, void* dW, int64_t lddw, float* dbias)
{
    S2V_ENTER(ctx);
    const auto bad = [&](int status, const char* what) { return s2v_fail(ctx, status, std::string("linear_i8_grad: ") + what); };
    if (m < 0 || n < 0 || k < 1) return bad(S2V_ERR_INVALID_ARG, "negative size or no columns");
    if (!s2v_dtype_ok(dy_type)) return bad(S2V_ERR_INVALID_ARG, "unknown element type");
    if (n == 0) return S2V_OK;
    if (m > INT32_MAX || n > INT32_MAX || k > INT32_MAX || !mm16_size_ok(m, n) || !mm16_size_ok(m, k) || !mm16_size_ok(n, k))
        return bad(S2V_ERR_UNSUPPORTED, "a size above 2^31 - 1, or a matrix above 2^56 numbers");
    const int64_t es = (int64_t)s2v_dtype_bytes(dy_type);
    if (!dW || (m > 0 && (!dy || !q || !q_scale))) return bad(S2V_ERR_INVALID_ARG, "NULL pointer");
    if ((m > 1 && (lddy < n || ldq < k)) || (n > 1 && lddw < k)) return bad(S2V_ERR_INVALID_ARG, "leading dimension below the number of columns");
    if (reinterpret_cast<uintptr_t>(dy) % es || reinterpret_cast<uintptr_t>(dW) % es || !s2v_aligned4(q_scale, dbias)) return bad(S2V_ERR_INVALID_ARG, "misaligned pointer");
    if (workspace_bytes < s2v_linear_i8_grad_workspace_bytes(m, n, k, dy_type) || (!workspace && workspace_bytes)) return bad(S2V_ERR_WORKSPACE, "workspace too small");
    if (!s2v_aligned16(workspace)) return bad(S2V_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    if (m == 0) {   // empty sums
        S2V_CUDA_OK(ctx, cudaMemset2DAsync(dW, (size_t)(n > 1 ? lddw : k) * es, 0, (size_t)k * es, (size_t)n, st));
        if (dbias) S2V_CUDA_OK(ctx, cudaMemsetAsync(dbias, 0, (size_t)n * sizeof(float), st));
        return S2V_OK;
    }
    if (m <= LG_FEW && n <= LG_FEW_PRODUCTS / m / k && (n + 63) / 64 <= 65535)
        return s2v_by_dtype(dy_type, [&](auto type) {
            using T = decltype(type);
            grad_few_kernel<T><<<dim3((unsigned)((k + 255) / 256), (unsigned)((n + 63) / 64)), 256, 0, st>>>((int)m, n, k, static_cast<const T*>(dy), lddy, q, ldq, q_scale, static_cast<T*>(dW),
                                                                                                            lddw, dbias);
            S2V_CHECK_LAUNCH(ctx, "grad_few_kernel");
            return (int)S2V_OK;
        });
    unsigned char* const ws = mm16_space(workspace);
    const bool direct = linear_i8_direct_takes(m, n, k, dy_type) && linear_i8_direct_lies(m, dy_type, dy, lddy, q, ldq);
    const LgSpace space(m, n, k, dy_type, direct);
    float* const columns = reinterpret_cast<float*>(ws + space.columns);
    float* const factor = dy_type == S2V_F16 ? reinterpret_cast<float*>(ws + space.factor) : nullptr;
    LgRows r{m, n, lddy, 0, dy, q_scale, nullptr, s2v_aligned16(dy) && (m <= 1 || lddy * es % 16 == 0), 1, reinterpret_cast<uint16_t*>(ws + space.dy), space.ldn, space.piece * space.ldn, columns};
    while (r.groups < 32 && r.groups * 8 < n) r.groups *= 2;
    const int64_t blocks = (n + r.groups * 8 - 1) / (r.groups * 8), lanes = LG_THREADS / r.groups;
    // `rows` of r in at most `most` shares; how many there are
    const auto shared_out = [&](int64_t rows, int64_t most) {
        const int64_t slabs = std::max<int64_t>(1, std::min({most, (8 * (int64_t)ctx->sm_count + blocks - 1) / blocks, (rows + 4 * lanes - 1) / (4 * lanes)}));
        r.m = rows, r.share = (rows + slabs - 1) / slabs;
        return (rows + r.share - 1) / r.share;
    };
    const auto lines = [&](auto kernel, int64_t count, float* out) {
        kernel<<<(unsigned)((n + 31) / 32), 256, 0, st>>>((int)count, n, columns, out);
        S2V_CHECK_LAUNCH(ctx, "grad_lines_kernel");
        return (int)S2V_OK;
    };
    if (factor) {
        const int64_t slabs = shared_out(m, LG_SLABS);
        grad_rows_kernel<__half, false><<<dim3((unsigned)blocks, (unsigned)slabs), LG_THREADS, 0, st>>>(r);
        S2V_CHECK_LAUNCH(ctx, "grad_rows_kernel");
        const int rc = lines(grad_lines_kernel<false>, slabs, factor);
        if (rc != S2V_OK) return rc;
        r.factor = factor;
    }
    if (direct) {
        const linear_i8_grad_args d{m, n, k, lddy, ldq, lddw, dy_type, dy, q, q_scale, factor, factor ? factor + n : nullptr, dW};
        int shares = 0;
        const int rc = linear_i8_direct(ctx, st, d, reinterpret_cast<float*>(ws + space.lines), dbias ? columns : nullptr, &shares);
        return rc == S2V_OK && dbias ? lines(grad_lines_kernel<true>, shares, dbias) : rc;
    }
    mm16_args g;
    g.type = dy_type == S2V_F16 ? S2V_F16 : S2V_BF16;
    g.a.p = ws + space.dy, g.a.cols = n, g.a.ld = space.ldn, g.a.part = r.part, g.a.parts = (int)space.parts;
    g.b.p = ws + space.q, g.b.cols = k, g.b.ld = space.ldk;
    g.m = n, g.n = k;
    g.alpha = factor ? factor + n : nullptr, g.alpha_rows = 1;
    g.lines = reinterpret_cast<float*>(ws + space.lines), g.sum = reinterpret_cast<float*>(ws + space.sum);
    g.out_type = dy_type, g.ldo = lddw;
    int64_t all_lines = 0;
    for (int64_t first = 0; first < m; first += space.piece) {
        const int64_t rows = std::min(space.piece, m - first), slabs = shared_out(rows, space.slabs);
        r.dy = static_cast<const unsigned char*>(dy) + (size_t)first * (m > 1 ? lddy : 0) * es, r.scale = q_scale + first, r.lines = columns + all_lines * n;
        all_lines += slabs;
        int rc = s2v_by_dtype(dy_type, [&](auto type) {
            grad_rows_kernel<decltype(type), true><<<dim3((unsigned)blocks, (unsigned)slabs), LG_THREADS, 0, st>>>(r);
            S2V_CHECK_LAUNCH(ctx, "grad_rows_kernel");
            return (int)S2V_OK;
        });
        if (rc != S2V_OK) return rc;
        const int64_t units = (rows * (space.ldk / 8) + 255) / 256, cap = 32 * (int64_t)ctx->sm_count;
        const int wide = reinterpret_cast<uintptr_t>(q) % 8 == 0 && (m <= 1 || ldq % 8 == 0);
        const auto kernel = dy_type == S2V_F16 ? grad_q_kernel<__half> : grad_q_kernel<__nv_bfloat16>;
        kernel<<<(unsigned)(units < cap ? units : cap), 256, 0, st>>>(rows, k, q + (size_t)first * (m > 1 ? ldq : 0), ldq, wide, reinterpret_cast<uint16_t*>(ws + space.q), space.ldk);
        S2V_CHECK_LAUNCH(ctx, "grad_q_kernel");
        g.a.rows = g.b.rows = g.k = rows, g.add = first > 0;
        if (first + rows == m) g.out = dW;
        rc = mm16_launch(ctx, st, MM16_OUT_ACROSS, g);
        if (rc != S2V_OK) return rc;
    }
    return dbias ? lines(grad_lines_kernel<true>, all_lines, dbias) : (int)S2V_OK;
}

}  // extern "C"
