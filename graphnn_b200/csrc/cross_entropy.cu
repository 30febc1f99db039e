// Softmax cross entropy of z = x W^T against a class a row, and its gradients, without z in memory:
//     loss_i = w_i log sum_j exp(z_ij - z_it),   G_ij = w_i (exp(z_ij - lse_i) - [j = t_i]),   dx = G W,   dW = G^T x.
// A pass over W leaves, for every row and tile of classes, the largest logit m and l = sum exp(z - m) of the classes other than the row's own, and the row's own
// logit; joined, they give log sum_j exp(z_ij - z_it) = log1p(sum of the others relative to the own class), which keeps its digits where the own class has
// nearly all of the probability.  The gradient computes the logits again, a piece of the vocabulary at a time, and multiplies the piece's G.
#include "product_simt.cuh"

namespace
{

constexpr int XE_TILE = PS_TILE;                  // classes of a partial sum
constexpr size_t XE_PIECE = (size_t)64 << 20;     // bytes of G, about

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

struct xe_rows {
    const int32_t* target;
    const float* weight;   // NULL: ones
    int64_t vocab;
    // the row's class, -1 if it is left out
    __device__ __forceinline__ int64_t own(int64_t i) const
    {
        const int64_t t = target[i];
        return t < 0 || t >= vocab || (weight && weight[i] == 0.0f) ? -1 : t;
    }
};

// rows of x, zeros where the row is left out
template <typename T> struct xe_x_across_k {
    static constexpr bool K_FAST = false;
    const T* p;
    int64_t ld;
    xe_rows rows;
    __device__ __forceinline__ float operator()(int64_t i, int64_t k) const { return rows.own(k) < 0 ? 0.0f : to_f32(p[k * ld + i]); }
};

struct xe_partials {   // 16 threads a row of the tile
    int64_t rows_n, vocab;
    xe_rows rows;
    float2* part;      // [tiles of classes][rows]
    float* mine;       // [rows]: the own class's logit
    __device__ __forceinline__ void operator()(int64_t r0, int64_t c0, const float (&acc)[4][4]) const
    {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t i = r0 + r, own = i < rows_n ? rows.own(i) : -1;
            xe_sum s{-INFINITY, 0.0f};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int64_t j = c0 + c;
                if (j >= vocab) continue;
                if (j == own) mine[i] = acc[r][c];
                else s.join(acc[r][c], 1.0f);
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
                const float mb = __shfl_xor_sync(0xffffffffu, s.m, o), lb = __shfl_xor_sync(0xffffffffu, s.l, o);
                s.join(mb, lb);
            }
            if (i < rows_n && (threadIdx.x & 15) == 0) part[c0 / XE_TILE * rows_n + i] = make_float2(s.m, s.l);
        }
    }
};

__global__ void __launch_bounds__(128) xe_join_kernel(int64_t rows_n, int tiles, xe_rows rows, const float2* __restrict__ part, const float* __restrict__ mine, float* __restrict__ loss,
                                                      float2* __restrict__ stats)
{
    const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (i >= rows_n) return;
    if (rows.own(i) < 0) {
        loss[i] = 0.0f;
        if (stats) stats[i] = make_float2(0.0f, 0.0f);
        return;
    }
    xe_sum s{-INFINITY, 0.0f};
    for (int t = 0; t < tiles; ++t) {
        const float2 p = part[(int64_t)t * rows_n + i];
        s.join(p.x, p.y);
    }
    // log(1 + l exp(m - z_t)), from whichever side is the larger
    const double d = (double)s.m - (double)mine[i];
    const double one = s.m == -INFINITY && s.l == 0.0f ? (mine[i] - mine[i]) : d > 0 ? d + log((double)s.l + exp(-d)) : log1p((double)s.l * exp(d));
    loss[i] = (float)(one * (rows.weight ? (double)rows.weight[i] : 1.0));
    if (stats) stats[i] = make_float2((float)(one + (double)mine[i]), (float)expm1(-one));
}

struct xe_gradient {   // a piece's G
    int64_t rows_n, cols, first;   // the piece's classes: first to first + cols
    xe_rows rows;
    const float2* stats;
    float* g;
    int64_t ldg;
    __device__ __forceinline__ void operator()(int64_t r0, int64_t c0, const float (&acc)[4][4]) const
    {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t i = r0 + r;
            if (i >= rows_n) continue;
            const int64_t own = rows.own(i);
            const float w = own < 0 ? 0.0f : rows.weight ? rows.weight[i] : 1.0f;
            const float2 st = stats[i];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (c0 + c < cols) g[i * ldg + c0 + c] = own < 0 ? 0.0f : w * (first + c0 + c == own ? st.y : expf(acc[r][c] - st.x));
        }
    }
};

// outputs added to those of the pieces before
template <typename T> struct xe_add_outputs {
    float* sum;
    T* p;   // NULL before the last piece
    int64_t ld, m, n;
    int start;
    __device__ __forceinline__ void operator()(int64_t r0, int64_t c0, const float (&acc)[4][4]) const
    {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (r0 + r < m && c0 + c < n) {
                    float* const s = sum + (r0 + r) * n + c0 + c;
                    const float v = start ? acc[r][c] : *s + acc[r][c];
                    if (p) p[(r0 + r) * ld + c0 + c] = from_f32<T>(v);
                    else *s = v;
                }
    }
};

// Where things lie in the workspace.
struct xe_space {
    size_t part = 0, mine = 0, g = 0, sum = 0, bytes = 0;
    int64_t piece = 0;
    xe_space(int64_t rows, int64_t vocab, int64_t k, bool grad)
    {
        const auto take = [&](size_t& at, size_t n) { at = bytes, bytes += (n + 255) / 256 * 256; };
        if (!grad) {
            take(mine, (size_t)rows * sizeof(float));
            take(part, (size_t)rows * (size_t)((vocab + XE_TILE - 1) / XE_TILE) * sizeof(float2));
            return;
        }
        piece = (int64_t)(XE_PIECE / sizeof(float)) / rows / XE_TILE * XE_TILE;
        piece = piece < XE_TILE ? XE_TILE : piece > vocab ? vocab : piece;
        take(g, (size_t)rows * (size_t)piece * sizeof(float));
        take(sum, (size_t)rows * (size_t)k * sizeof(float));
    }
};

int check(s2v_ctx* ctx, const char* name, int64_t rows, int64_t vocab, int64_t k, int type, const void* x, int64_t ldx, const void* W, int64_t ldw, const int32_t* target,
          const float* row_weight)
{
    const auto bad = [&](int status, const char* what) { return s2v_fail(ctx, status, std::string(name) + ": " + what); };
    if (rows < 0 || vocab < 1 || k < 1) return bad(S2V_ERR_INVALID_ARG, "negative size, or no classes or no columns");
    if (!s2v_dtype_ok(type)) return bad(S2V_ERR_INVALID_ARG, "unknown element type");
    if (rows > INT32_MAX || vocab > INT32_MAX || k > INT32_MAX) return bad(S2V_ERR_UNSUPPORTED, "a size above 2^31 - 1");
    if (rows == 0) return S2V_OK;
    if (!x || !W || !target) return bad(S2V_ERR_INVALID_ARG, "NULL pointer");
    if ((rows > 1 && ldx < k) || (vocab > 1 && ldw < k)) return bad(S2V_ERR_INVALID_ARG, "leading dimension below the number of columns");
    const size_t es = s2v_dtype_bytes(type);
    if (reinterpret_cast<uintptr_t>(x) % es || reinterpret_cast<uintptr_t>(W) % es || !s2v_aligned4(target, row_weight)) return bad(S2V_ERR_INVALID_ARG, "misaligned pointer");
    return S2V_OK;
}

}  // namespace

extern "C" {

size_t s2v_linear_cross_entropy_workspace_bytes(int64_t rows, int64_t vocab, int64_t k, int type, int grad)
{
    if (rows <= 0 || vocab <= 0 || k <= 0 || rows > INT32_MAX || vocab > INT32_MAX || k > INT32_MAX || !s2v_dtype_ok(type)) return 0;
    const size_t loss = xe_space(rows, vocab, k, false).bytes;
    const size_t both = grad ? xe_space(rows, vocab, k, true).bytes : 0;
    return loss > both ? loss : both;
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
    const xe_space space(rows, vocab, k, false);
    if (!workspace || workspace_bytes < s2v_linear_cross_entropy_workspace_bytes(rows, vocab, k, type, 0)) return bad(S2V_ERR_WORKSPACE, "workspace too small");
    if (!s2v_aligned16(workspace)) return bad(S2V_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    unsigned char* const ws = static_cast<unsigned char*>(workspace);
    float2* const part = reinterpret_cast<float2*>(ws + space.part);
    float* const mine = reinterpret_cast<float*>(ws + space.mine);
    const xe_rows r{target, row_weight, vocab};
    const int done = s2v_by_dtype(type, [&](auto t) {
        using T = decltype(t);
        return product_simt(ctx, st, "linear_cross_entropy", rows, vocab, k, along_k<T>{static_cast<const T*>(x), ldx}, along_k<T>{static_cast<const T*>(W), ldw},
                            xe_partials{rows, vocab, r, part, mine});
    });
    if (done != S2V_OK) return done;
    xe_join_kernel<<<(unsigned)((rows + 127) / 128), 128, 0, st>>>(rows, (int)((vocab + XE_TILE - 1) / XE_TILE), r, part, mine, loss, reinterpret_cast<float2*>(stats));
    S2V_CHECK_LAUNCH(ctx, "xe_join_kernel");
    return S2V_OK;
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
    const xe_space space(rows, vocab, k, true);
    if (!workspace || workspace_bytes < s2v_linear_cross_entropy_workspace_bytes(rows, vocab, k, type, 1)) return bad(S2V_ERR_WORKSPACE, "workspace too small");
    if (!s2v_aligned16(workspace)) return bad(S2V_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
    unsigned char* const ws = static_cast<unsigned char*>(workspace);
    float* const g = reinterpret_cast<float*>(ws + space.g);
    float* const sum = reinterpret_cast<float*>(ws + space.sum);
    const xe_rows r{target, row_weight, vocab};
    return s2v_by_dtype(type, [&](auto t) {
        using T = decltype(t);
        const T* const xt = static_cast<const T*>(x);
        const T* const wt = static_cast<const T*>(W);
        for (int64_t first = 0; first < vocab; first += space.piece) {
            const int64_t cols = space.piece < vocab - first ? space.piece : vocab - first;
            int done = product_simt(ctx, st, "linear_cross_entropy_grad", rows, cols, k, along_k<T>{xt, ldx}, along_k<T>{wt + first * ldw, ldw},
                                    xe_gradient{rows, cols, first, r, reinterpret_cast<const float2*>(stats), g, space.piece});
            if (done == S2V_OK && dx)
                done = product_simt(ctx, st, "linear_cross_entropy_grad", rows, k, cols, along_k<float>{g, space.piece}, across_k<T>{wt + first * ldw, ldw},
                                    xe_add_outputs<T>{sum, first + cols == vocab ? static_cast<T*>(dx) : nullptr, lddx, rows, k, first == 0});
            if (done == S2V_OK && dW)
                done = product_simt(ctx, st, "linear_cross_entropy_grad", cols, k, rows, across_k<float>{g, space.piece}, xe_x_across_k<T>{xt, ldx, r},
                                    store_outputs<T>{static_cast<T*>(dW) + first * lddw, lddw, cols, k});
            if (done != S2V_OK) return done;
        }
        return (int)S2V_OK;
    });
}

}  // extern "C"
