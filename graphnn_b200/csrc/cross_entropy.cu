// Softmax cross entropy of z = x W^T against a class a row, and its gradients, without z in memory:
//     loss_i = w_i log sum_j exp(z_ij - z_it),   G_ij = w_i (exp(z_ij - lse_i) - [j = t_i]),   dx = G W,   dW = G^T x.
// A pass over W leaves, for every row and tile of classes, the largest logit m and l = sum exp(z - m) of the classes other than the row's own, and the row's own
// logit; joined, they give log sum_j exp(z_ij - z_it) = log1p(sum of the others relative to the own class), which keeps its digits where the own class has
// nearly all of the probability.  The gradient computes the logits again, a piece of the vocabulary at a time, leaves the piece's G in memory in 16 bits
// (what the tensor cores multiply; three parts of it where x and W are fp32) and multiplies it.  G in 16 bits is off by half a step of them, as x and W are.
//
// Where the logits are few and their sums long, tiles of logits would leave most of the GPU idle: then k is shared out, and the logits, a few MB of fp32, go through memory.
#include <algorithm>

#include "cross_entropy_few.cuh"
#include "cross_entropy_rows.cuh"
#include "mm16.cuh"

namespace
{

constexpr size_t XE_G_BYTES = (size_t)256 << 20;      // of a piece's G
constexpr size_t XE_W_BYTES = (size_t)128 << 20;      // of a piece of W that has to be copied
constexpr size_t XE_PART_BYTES = (size_t)256 << 20;   // of a piece's partial sums
constexpr int64_t XE_TILE = 256;                      // pieces are multiples of it

// a sum of exponentials, l * exp(m)
struct xe_sum {
    float m, l;
    __device__ __forceinline__ void join(float mb, float lb)
    {
        const float top = fmaxf(m, mb);
        if (top == -INFINITY && lb == lb && l == l) return;   // nothing on either side
        const float from = top == INFINITY ? 0.0f : top;
        l = l * expf(m - from) + lb * expf(mb - from);
        m = top;
    }
};

// The partial sums of a piece, THREADS threads a row, onto what the pieces before gave (`run`, [rows]; first: nothing yet); after the last piece the loss.
template <int THREADS>
__global__ void __launch_bounds__(256) xe_join_kernel(int64_t rows_n, int lines, xe_rows rows, const float2* __restrict__ part, const float* __restrict__ mine, float2* __restrict__ run, int first,
                                                      int last, float* __restrict__ loss, float2* __restrict__ stats)
{
    constexpr int ROWS = 256 / THREADS;
    __shared__ float2 of[THREADS][ROWS];
    const int at = threadIdx.x % ROWS, g = threadIdx.x / ROWS;
    const int64_t i = (int64_t)blockIdx.x * ROWS + at;
    xe_sum s{-INFINITY, 0.0f};
    if (i < rows_n)
        for (int t = g; t < lines; t += 4 * THREADS) {
            float2 p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) p[u] = t + u * THREADS < lines ? part[(int64_t)(t + u * THREADS) * rows_n + i] : make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int u = 0; u < 4; ++u) s.join(p[u].x, p[u].y);
        }
    of[g][at] = make_float2(s.m, s.l);
    __syncthreads();
#pragma unroll
    for (int o = THREADS / 2; o; o >>= 1) {
        if (g < o) {
            s.join(of[g + o][at].x, of[g + o][at].y);
            of[g][at] = make_float2(s.m, s.l);
        }
        __syncthreads();
    }
    if (g || i >= rows_n) return;
    if (!first) s.join(run[i].x, run[i].y);
    if (!last) {
        run[i] = make_float2(s.m, s.l);
        return;
    }
    if (rows.its(i) < 0) {
        loss[i] = 0.0f;
        if (stats) stats[i] = make_float2(0.0f, 0.0f);
        return;
    }
    xe_finish(rows, i, s.m, s.l, mine[i], loss, stats);
}
int xe_join(s2v_ctx* ctx, cudaStream_t st, int64_t rows_n, int lines, xe_rows rows, const float2* part, const float* mine, float2* run, bool first, bool last, float* loss, float* stats)
{
    const auto go = [&](auto kernel, int threads) {
        const int64_t per = 256 / threads;
        kernel<<<(unsigned)((rows_n + per - 1) / per), 256, 0, st>>>(rows_n, lines, rows, part, mine, run, first, last, loss, reinterpret_cast<float2*>(stats));
        S2V_CHECK_LAUNCH(ctx, "xe_join_kernel");
        return (int)S2V_OK;
    };
    // (one row of 2048 lines by 64 threads 10 us)
    return rows_n >= 2048 || lines <= 32 ? go(xe_join_kernel<8>, 8) : rows_n > 64 ? go(xe_join_kernel<64>, 64) : go(xe_join_kernel<256>, 256);
}

// G in 16 bits is held relative to the largest row weight (times `unit`, 2^14 for fp16, whose smallest step is then 2^-38 of that weight): where all rows weigh the same, which
// is the rule, the own class's G of a row that does not know it is next to -1, and rounds to it, instead of all such rows being rounded alike by what that weight is
// off in 16 bits (4096 x 131072 x 4096 bf16: dW 2.6e-3 off for one number of rows, 2.0e-3 for another).  Rows of smaller weights are rounded as any number is, half a step of 16 bits (2048 rows of
// weights 0.2 to 1.2, 4000 classes, k = 64, bf16: what G's rounding adds to dW is 1.4e-3 of it, with one weight 3.9e-4; rounding dW itself 1.7e-3).  factor[0], and factor[1] = 1 / factor[0].
__global__ void __launch_bounds__(1024) xe_factor_kernel(int64_t rows_n, xe_rows rows, float unit, float* factor)
{
    __shared__ uint32_t part[32];
    uint32_t top = 0;
    for (int64_t i = threadIdx.x; i < rows_n; i += 1024)
        if (rows.own(i) >= 0) {
            const uint32_t w = rows.weight ? __float_as_uint(rows.weight[i]) & 0x7fffffffu : 0x3f800000u;
            if (w < 0x7f800000u) top = max(top, w);
        }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    top = __reduce_max_sync(0xffffffffu, part[threadIdx.x]);
    if (threadIdx.x == 0) {
        const float largest = fminf(fmaxf(__uint_as_float(top), 7.888609052210118e-31f), 1.2676506002282294e30f);   // (2^-100 to 2^100: weights outside are not scaled further)
        factor[0] = unit / largest, factor[1] = largest / unit;
    }
}

// What a row's G is multiplied by before it is rounded to 16 bits, and what the rounding takes from the own class's, a row's largest number by far: dx gets that
// times the class's row of W back, in fp32 (400 rows, 5000 classes, fp16: 1.4e-4 off from the rounding of G without it, relative, 2e-5 with it; bf16 1.0e-3 and 1.6e-4).
template <typename H> __global__ void __launch_bounds__(256) xe_row_scale_kernel(int64_t rows_n, xe_rows rows, const float2* __restrict__ stats, const float* __restrict__ factor,
                                                                                 float* __restrict__ scale, float* __restrict__ fix)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows_n) return;
    float s = 0.0f, f = 0.0f;
    if (rows.own(i) >= 0) {
        s = (rows.weight ? rows.weight[i] : 1.0f) * (factor ? factor[0] : 1.0f);
        const float own = s * stats[i].y;
        f = (own - to_f32(from_f32<H>(own))) * (factor ? factor[1] : 1.0f);
    }
    scale[i] = s, fix[i] = f;
}

// Few logits, long sums: at most half of 148 tiles, and 32 panels or more of each (86 x 38 x 3206 fp32, a step: 270 us with whole tiles).
bool xe_keeps(int64_t rows, int64_t vocab, int64_t k, int parts)
{
    return ((rows + 127) / 128) * ((vocab + 127) / 128) <= 74 && (k + 63) / 64 * (parts == 3 ? 6 : 1) >= 32;
}
// The loss from a row of logits, a row a CTA
__global__ void __launch_bounds__(256) xe_kept_loss_kernel(xe_rows rows, const float* __restrict__ z, int64_t ldz, float* __restrict__ loss, float2* __restrict__ stats)
{
    __shared__ float of[2][8];
    const int64_t i = blockIdx.x, own = stats ? rows.its(i) : rows.own(i);
    if (own < 0) {
        if (threadIdx.x == 0) {
            loss[i] = 0.0f;
            if (stats) stats[i] = make_float2(0.0f, 0.0f);
        }
        return;
    }
    const float* const row = z + i * ldz;
    float top = -INFINITY;   // of the other classes
    for (int64_t j = threadIdx.x; j < rows.vocab; j += 256)
        if (j != own) top = fmaxf(top, row[j]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) of[0][threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, of[0][w]);
    const float from = fabsf(top) == INFINITY ? 0.0f : top;
    float l = 0.0f;
    for (int64_t j = threadIdx.x; j < rows.vocab; j += 256)
        if (j != own) l += top == INFINITY ? NAN : expf(row[j] - from);
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if ((threadIdx.x & 31) == 0) of[1][threadIdx.x >> 5] = l;
    __syncthreads();
    if (threadIdx.x) return;
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) l += of[1][w];
    xe_finish(rows, i, top, l, row[own], loss, stats);
}
// A piece's G from kept logits, in 16-bit parts, eight classes a thread
template <typename H> __global__ void __launch_bounds__(256) xe_kept_grad_kernel(int64_t rows_n, int64_t cols, int64_t first, xe_rows rows, const float* __restrict__ z, int64_t ldz,
                                                                                 const float2* __restrict__ stats, const float* __restrict__ row_scale, uint16_t* __restrict__ g, int64_t ldg,
                                                                                 int64_t part, int parts)
{
    const int64_t per_row = (cols + 7) / 8, all = rows_n * per_row;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < all; at += (int64_t)gridDim.x * 256) {
        const int64_t i = at / per_row, c = (at - i * per_row) * 8, own = rows.own(i) - first;
        const float w = row_scale[i];
        const float2 st = stats[i];
        const float* const row = z + i * ldz + first + c;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = w == 0.0f || c + e >= cols ? 0.0f : w * (c + e == own ? st.y : expf(row[e] - st.x));
        for (int p = 0; p < parts; ++p) {
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h[j] = pack_16bit<H>(y[2 * j], y[2 * j + 1]);
                if constexpr (std::is_same<H, __nv_bfloat16>::value) y[2 * j] -= __uint_as_float(h[j] << 16), y[2 * j + 1] -= __uint_as_float(h[j] & 0xffff0000u);
            }
            *reinterpret_cast<uint4*>(g + p * part + i * ldg + c) = make_uint4(h[0], h[1], h[2], h[3]);
        }
    }
}

// Where things lie in the workspace, and how many classes a piece has.  `copied`: whether W has to be copied (fp32, or rows that don't lie on 16-byte boundaries).
struct xe_space {
    size_t mine = 0, run = 0, part = 0, x16 = 0, w16 = 0, factor = 0, scale = 0, g = 0, sum = 0, lines = 0, z = 0, bytes = 0;
    bool keeps;
    int64_t ldz = 0, piece = 0, ld16 = 0, ldg = 0, parts = 0;
    xe_space(int64_t rows, int64_t vocab, int64_t k, int type, bool grad, bool copied)
    {
        const auto take = [&](size_t& at, size_t n) { at = bytes, bytes += (n + 255) / 256 * 256; };
        parts = type == S2V_F32 ? 3 : 1;
        ld16 = (k + 7) / 8 * 8, ldz = mm16_pitch(vocab);
        keeps = xe_keeps(rows, vocab, k, (int)parts);
        const int products = parts == 3 ? 6 : 1;
        if (keeps) take(z, (size_t)rows * ldz * sizeof(float));
        const auto of = [&](size_t all, size_t each) { return std::max((int64_t)(all / each) / XE_TILE * XE_TILE, XE_TILE); };
        piece = vocab;
        if (copied) piece = std::min(piece, of(XE_W_BYTES, (size_t)ld16 * 2 * parts));
        if (grad) {
            piece = std::min(piece, of(XE_G_BYTES, (size_t)rows * 2 * parts));
            ldg = (piece + 63) / 64 * 64;
            take(factor, 2 * sizeof(float));
            take(scale, 2 * (size_t)rows * sizeof(float));
            take(g, (size_t)rows * ldg * 2 * parts);
            take(sum, (size_t)rows * mm16_pitch(k) * sizeof(float));
            take(lines, std::max({mm16_lines_bytes(piece, products), mm16_lines_bytes(rows, products), keeps ? mm16_lines_bytes(k, products) : 0}));
        } else if (keeps) take(lines, mm16_lines_bytes(k, products));
        else {
            piece = std::min(piece, of(XE_PART_BYTES, (size_t)rows * sizeof(float2)) * 64);   // (a line for every 64 classes at most)
            take(mine, (size_t)rows * sizeof(float));
            take(run, (size_t)rows * sizeof(float2));
            take(part, (size_t)rows * mm16_sum_lines_most(piece) * sizeof(float2));
        }
        if (copied) take(w16, (size_t)piece * ld16 * 2 * parts);
        take(x16, (size_t)rows * ld16 * 2 * parts);
    }
};

int check(s2v_ctx* ctx, const char* name, int64_t rows, int64_t vocab, int64_t k, int type, const void* x, int64_t ldx, const void* W, int64_t ldw, const int32_t* target,
          const float* row_weight)
{
    const auto bad = [&](int status, const char* what) { return s2v_fail(ctx, status, std::string(name) + ": " + what); };
    if (rows < 0 || vocab < 1 || k < 1) return bad(S2V_ERR_INVALID_ARG, "negative size, or no classes or no columns");
    if (!s2v_dtype_ok(type)) return bad(S2V_ERR_INVALID_ARG, "unknown element type");
    if (rows > INT32_MAX || vocab > INT32_MAX || k > INT32_MAX || !mm16_size_ok(rows, k) || !mm16_size_ok(vocab, k))
        return bad(S2V_ERR_UNSUPPORTED, "a size above 2^31 - 1, or a matrix above 2^56 numbers");
    if (rows == 0) return S2V_OK;
    if (!x || !W || !target) return bad(S2V_ERR_INVALID_ARG, "NULL pointer");
    if ((rows > 1 && ldx < k) || (vocab > 1 && ldw < k)) return bad(S2V_ERR_INVALID_ARG, "leading dimension below the number of columns");
    const size_t es = s2v_dtype_bytes(type);
    if (reinterpret_cast<uintptr_t>(x) % es || reinterpret_cast<uintptr_t>(W) % es || !s2v_aligned4(target, row_weight)) return bad(S2V_ERR_INVALID_ARG, "misaligned pointer");
    return S2V_OK;
}

// What both calls hand to the products: x and W in 16-bit parts, where they lie or copied.
struct xe_call {
    s2v_ctx* ctx;
    cudaStream_t st;
    bool copy_x, copy_w;
    xe_space space;
    xe_rows rows;
    mm16_args args;
    const unsigned char* W;
    int64_t ldw;
    int type;
    unsigned char* ws;
    unsigned char* w16;
    static bool lies(int type, const void* p, int64_t rows, int64_t ld) { return type != S2V_F32 && s2v_aligned16(p) && (rows <= 1 || ld % 8 == 0); }
    xe_call(s2v_ctx* ctx_, cudaStream_t st_, int64_t n, int64_t vocab, int64_t k, int type_, const void* x, int64_t ldx, const void* W_, int64_t ldw_, const int32_t* target, const float* weight,
            unsigned char* ws_, bool grad)
        : ctx(ctx_), st(st_), copy_x(grad || !lies(type_, x, n, ldx)), copy_w(!lies(type_, W_, vocab, ldw_)), space(n, vocab, k, type_, grad, copy_w), rows{target, weight, vocab},
          W(static_cast<const unsigned char*>(W_)), ldw(ldw_), type(type_), ws(ws_), w16(ws + space.w16)
    {
        args.type = type == S2V_F16 ? S2V_F16 : S2V_BF16;
        args.m = n, args.k = k;
        args.a.p = copy_x ? ws + space.x16 : x, args.a.rows = n, args.a.cols = k, args.a.ld = copy_x ? space.ld16 : ldx, args.a.part = n * space.ld16, args.a.parts = (int)space.parts;
        args.target = target, args.weight = weight, args.vocab = vocab;
    }
    // a piece's logits to memory
    int logits(mm16_args a, int64_t first) const
    {
        a.lines = reinterpret_cast<float*>(ws + space.lines);
        a.out = reinterpret_cast<float*>(ws + space.z) + first, a.out_type = S2V_F32, a.ldo = space.ldz;
        return mm16_launch(ctx, st, MM16_OUT_ALONG, a);
    }
    int piece_of_w(mm16_operand& b, int64_t first, int64_t cols) const
    {
        const unsigned char* const from = W + (size_t)first * (rows.vocab > 1 ? ldw : 0) * s2v_dtype_bytes(type);
        b.rows = cols, b.cols = args.k, b.parts = (int)space.parts;
        b.p = copy_w ? w16 : from, b.ld = copy_w ? space.ld16 : ldw, b.part = cols * space.ld16;
        return copy_w ? mm16_pack(ctx, st, cols, args.k, type, from, ldw, nullptr, nullptr, 0, w16, space.ld16, b.part) : S2V_OK;
    }
};

}  // namespace

extern "C" {

size_t s2v_linear_cross_entropy_workspace_bytes(int64_t rows, int64_t vocab, int64_t k, int type, int grad)
{
    if (rows <= 0 || vocab <= 0 || k <= 0 || rows > INT32_MAX || vocab > INT32_MAX || k > INT32_MAX || !s2v_dtype_ok(type)) return 0;
    if (!mm16_size_ok(rows, k) || !mm16_size_ok(vocab, k)) return 0;
    if (xe_few_takes(rows, vocab, k)) return xe_few_bytes(rows, vocab);
    size_t most = 0;   // wherever the matrices lie
    for (int form = 0; form < (grad ? 4 : 2); ++form)
        if ((form & 1) || type != S2V_F32) most = std::max(most, xe_space(rows, vocab, k, type, form & 2, form & 1).bytes);
    return most + MM16_SLACK;
}

int s2v_linear_cross_entropy(s2v_ctx* ctx, s2v_stream stream, int64_t rows, int64_t vocab, int64_t k, int type, const void* x, int64_t ldx, const void* W, int64_t ldw,
                             const int32_t* target, const float* row_weight, void* workspace, size_t workspace_bytes, float* loss, float* stats)
{
    S2V_ENTER(ctx);
    const int rc = check(ctx, "linear_cross_entropy", rows, vocab, k, type, x, ldx, W, ldw, target, row_weight);
    if (rc != S2V_OK || rows == 0) return rc;
    const auto bad = [&](int status, const char* what) { return s2v_fail(ctx, status, std::string("linear_cross_entropy: ") + what); };
    if (!loss) return bad(S2V_ERR_INVALID_ARG, "NULL pointer");
    if (!s2v_aligned4(loss) || reinterpret_cast<uintptr_t>(stats) % 8) return bad(S2V_ERR_INVALID_ARG, "misaligned pointer");
    if (!workspace || workspace_bytes < s2v_linear_cross_entropy_workspace_bytes(rows, vocab, k, type, 0)) return bad(S2V_ERR_WORKSPACE, "workspace too small");
    if (!s2v_aligned16(workspace)) return bad(S2V_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    if (xe_few_takes(rows, vocab, k)) return xe_few_loss(ctx, st, rows, vocab, k, type, x, ldx, W, ldw, target, row_weight, loss, stats);
    unsigned char* const ws = mm16_space(workspace);
    const xe_call c(ctx, st, rows, vocab, k, type, x, ldx, W, ldw, target, row_weight, ws, false);
    const xe_space& space = c.space;
    mm16_args a = c.args;
    a.weight = nullptr;   // (a row whose weight is 0 here may have another one in the gradient)
    int done = S2V_OK;
    if (c.copy_x) done = mm16_pack(ctx, st, rows, k, type, x, ldx, nullptr, nullptr, 0, ws + space.x16, space.ld16, rows * space.ld16);
    a.part = reinterpret_cast<float2*>(ws + space.part), a.mine = reinterpret_cast<float*>(ws + space.mine);
    for (int64_t first = 0; done == S2V_OK && first < vocab; first += space.piece) {
        const int64_t cols = std::min(space.piece, vocab - first);
        done = c.piece_of_w(a.b, first, cols);
        a.n = cols, a.first = first;
        if (space.keeps) {
            if (done == S2V_OK) done = c.logits(a, first);
            continue;
        }
        if (done == S2V_OK) done = mm16_launch(ctx, st, MM16_SUMS, a);
        if (done == S2V_OK)
            done = xe_join(ctx, st, rows, mm16_sum_lines(ctx, rows, cols), c.rows, a.part, a.mine, reinterpret_cast<float2*>(ws + space.run), first == 0, first + cols == vocab, loss, stats);
    }
    if (done == S2V_OK && space.keeps) {
        xe_kept_loss_kernel<<<(unsigned)rows, 256, 0, st>>>(c.rows, reinterpret_cast<const float*>(ws + space.z), space.ldz, loss, reinterpret_cast<float2*>(stats));
        S2V_CHECK_LAUNCH(ctx, "xe_kept_loss_kernel");
    }
    return done;
}

int s2v_linear_cross_entropy_grad(s2v_ctx* ctx, s2v_stream stream, int64_t rows, int64_t vocab, int64_t k, int type, const void* x, int64_t ldx, const void* W, int64_t ldw,
                                  const int32_t* target, const float* row_weight, const float* stats, void* workspace, size_t workspace_bytes, void* dx, int64_t lddx, void* dW,
                                  int64_t lddw)
{
    S2V_ENTER(ctx);
    const int rc = check(ctx, "linear_cross_entropy_grad", rows, vocab, k, type, x, ldx, W, ldw, target, row_weight);
    if (rc != S2V_OK) return rc;
    const auto bad = [&](int status, const char* what) { return s2v_fail(ctx, status, std::string("linear_cross_entropy_grad: ") + what); };
    const size_t es = s2v_dtype_bytes(type);
    if (reinterpret_cast<uintptr_t>(dx) % es || reinterpret_cast<uintptr_t>(dW) % es || reinterpret_cast<uintptr_t>(stats) % 8) return bad(S2V_ERR_INVALID_ARG, "misaligned pointer");
    if ((dx && rows > 1 && lddx < k) || (dW && vocab > 1 && lddw < k)) return bad(S2V_ERR_INVALID_ARG, "leading dimension below the number of columns");
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    if (rows == 0) {   // an empty sum
        if (dW) S2V_CUDA_OK(ctx, cudaMemset2DAsync(dW, (size_t)(vocab > 1 ? lddw : k) * es, 0, (size_t)k * es, (size_t)vocab, st));
        return S2V_OK;
    }
    if (!stats) return bad(S2V_ERR_INVALID_ARG, "NULL pointer");
    if (!dx && !dW) return S2V_OK;
    if (!workspace || workspace_bytes < s2v_linear_cross_entropy_workspace_bytes(rows, vocab, k, type, 1)) return bad(S2V_ERR_WORKSPACE, "workspace too small");
    if (!s2v_aligned16(workspace)) return bad(S2V_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
    if (xe_few_takes(rows, vocab, k)) return xe_few_grad(ctx, st, rows, vocab, k, type, x, ldx, W, ldw, target, row_weight, stats, workspace, dx, lddx, dW, lddw);
    unsigned char* const ws = mm16_space(workspace);
    const xe_call c(ctx, st, rows, vocab, k, type, x, ldx, W, ldw, target, row_weight, ws, true);
    const xe_space& space = c.space;
    // x with zeros in the rows that are left out, whatever these hold: their zeros of G meet zeros in dW
    int done = mm16_pack(ctx, st, rows, k, type, x, ldx, target, row_weight, vocab, ws + space.x16, space.ld16, rows * space.ld16);
    float* factor = nullptr;
    if (done == S2V_OK && type != S2V_F32) {
        factor = reinterpret_cast<float*>(ws + space.factor);
        xe_factor_kernel<<<1, 1024, 0, st>>>(rows, c.rows, type == S2V_F16 ? 16384.0f : 1.0f, factor);
        S2V_CHECK_LAUNCH(ctx, "xe_factor_kernel");
    }
    float* const scale = reinterpret_cast<float*>(ws + space.scale);
    const float2* const kept = reinterpret_cast<const float2*>(stats);
    if (done == S2V_OK) {
        const auto kernel = type == S2V_F32 ? xe_row_scale_kernel<float> : type == S2V_F16 ? xe_row_scale_kernel<__half> : xe_row_scale_kernel<__nv_bfloat16>;
        kernel<<<(unsigned)((rows + 255) / 256), 256, 0, st>>>(rows, c.rows, kept, factor, scale, scale + rows);
        S2V_CHECK_LAUNCH(ctx, "xe_row_scale_kernel");
    }
    mm16_args z = c.args;   // the logits again
    z.stats = kept, z.row_scale = scale;
    z.g = ws + space.g, z.ldg = space.ldg, z.g_part = rows * space.ldg, z.g_parts = (int)space.parts;
    for (int64_t first = 0; done == S2V_OK && first < vocab; first += space.piece) {
        const int64_t cols = std::min(space.piece, vocab - first);
        done = c.piece_of_w(z.b, first, cols);
        z.n = cols, z.first = first;
        if (done == S2V_OK) done = space.keeps ? c.logits(z, first) : mm16_launch(ctx, st, MM16_SOFTMAX_GRAD, z);
        if (done == S2V_OK && space.keeps) {
            const int64_t blocks = (rows * ((cols + 7) / 8) + 255) / 256;
            const auto kernel = type == S2V_F16 ? xe_kept_grad_kernel<__half> : xe_kept_grad_kernel<__nv_bfloat16>;
            kernel<<<(unsigned)blocks, 256, 0, st>>>(rows, cols, first, c.rows, reinterpret_cast<const float*>(ws + space.z), space.ldz, kept, scale, static_cast<uint16_t*>(z.g), space.ldg,
                                                     z.g_part, z.g_parts);
            S2V_CHECK_LAUNCH(ctx, "xe_kept_grad_kernel");
        }
        mm16_args p;
        p.type = z.type;
        p.a.p = z.g, p.a.rows = rows, p.a.cols = cols, p.a.ld = space.ldg, p.a.part = z.g_part, p.a.parts = (int)space.parts;
        p.alpha = factor ? factor + 1 : nullptr;
        p.lines = reinterpret_cast<float*>(ws + space.lines);
        p.out_type = type, p.n = k;
        if (done == S2V_OK && dx) {
            mm16_args q = p;
            q.b = z.b, q.m = rows, q.k = cols;
            q.sum = reinterpret_cast<float*>(ws + space.sum), q.add = first > 0;
            if (first + cols == vocab) {
                q.out = dx, q.ldo = lddx;
                if (type != S2V_F32) q.fix = scale + rows, q.target = target, q.vocab = vocab, q.fix_w = W, q.fix_ld = ldw;
            }
            done = mm16_launch(ctx, st, MM16_OUT, q);
        }
        if (done == S2V_OK && dW) {
            mm16_args q = p;
            q.b = z.a, q.m = cols, q.k = rows;
            q.out = static_cast<unsigned char*>(dW) + (size_t)first * (vocab > 1 ? lddw : k) * es, q.ldo = lddw;
            done = mm16_launch(ctx, st, MM16_OUT_ACROSS, q);
        }
    }
    return done;
}

}  // extern "C"
