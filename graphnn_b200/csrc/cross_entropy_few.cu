// Softmax cross entropy of z = x W^T and its gradients for up to 64 classes, 512 columns and 512 rows: fp32 arithmetic, one launch for the loss and two for the gradients.
// A warp has a row of x in registers, 32 columns apart a lane; a logit is a sum over the lanes, and stays with lane (class mod 32).
#include "cross_entropy_few.cuh"

namespace
{

constexpr int XF_CLASSES = 64, XF_COLS = 512, XF_ROWS = 512, XF_PER = XF_COLS / 32, XF_CTA = 128;

struct XfArgs {
    int rows, vocab, k;
    int64_t ldx, ldw, lddx, lddw;
    const void* x;
    const void* W;
    const int32_t* target;
    const float* weight;
    float* loss;
    float2* stats;
    float* g;   // [rows][vocab]
    void* dx;
    void* dW;
};

template <typename T> struct xf_row {
    float x[XF_PER];
    float z[XF_CLASSES / 32];   // of classes lane and lane + 32
    __device__ __forceinline__ xf_row(const XfArgs& a, int i)
    {
        const int lane = threadIdx.x & 31;
        const T* const from = static_cast<const T*>(a.x) + i * a.ldx;
#pragma unroll
        for (int u = 0; u < XF_PER; ++u) x[u] = lane + 32 * u < a.k ? to_f32(from[lane + 32 * u]) : 0.0f;
        z[0] = z[1] = -INFINITY;
        for (int j0 = 0; j0 < a.vocab; j0 += 4) {   // four sums at a time
            float s[4] = {};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const T* const w = static_cast<const T*>(a.W) + min(j0 + c, a.vocab - 1) * a.ldw;
#pragma unroll
                for (int u = 0; u < XF_PER; ++u)
                    if (lane + 32 * u < a.k) s[c] = fmaf(x[u], to_f32(w[lane + 32 * u]), s[c]);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[c] += __shfl_xor_sync(0xffffffffu, s[c], o);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (j0 + c < a.vocab && lane == ((j0 + c) & 31)) z[(j0 + c) >> 5] = s[c];
        }
    }
};

__device__ __forceinline__ int xf_own(const XfArgs& a, int i)
{
    const int t = a.target[i];
    return t < 0 || t >= a.vocab || (a.weight && a.weight[i] == 0.0f) ? -1 : t;
}

template <typename T> __global__ void __launch_bounds__(XF_CTA) xe_few_loss_kernel(const XfArgs a)
{
    const int i = blockIdx.x * (XF_CTA / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (i >= a.rows) return;
    const int own = xf_own(a, i);
    if (own < 0) {
        if (lane == 0) {
            a.loss[i] = 0.0f;
            if (a.stats) a.stats[i] = make_float2(0.0f, 0.0f);
        }
        return;
    }
    const xf_row<T> row(a, i);
    const float mine = __shfl_sync(0xffffffffu, own < 32 ? row.z[0] : row.z[1], own & 31);
    // the other classes' exponentials, relative to the own one's
    float top = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (lane + 32 * h != own) top = fmaxf(top, row.z[h]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float from = fabsf(top) == INFINITY ? 0.0f : top;
    float l = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int j = lane + 32 * h;
        if (j != own && j < a.vocab) l += top == INFINITY ? NAN : expf(row.z[h] - from);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane) return;
    const double d = (double)top - (double)mine;
    const double one = top == -INFINITY && l == 0.0f ? (double)(mine - mine) : d > 0 ? d + log((double)l + exp(-d)) : log1p((double)l * exp(d));
    a.loss[i] = (float)(one * (a.weight ? (double)a.weight[i] : 1.0));
    if (a.stats) a.stats[i] = make_float2((float)(one + (double)mine), (float)expm1(-one));
}

// G and dx, a row a warp
template <typename T> __global__ void __launch_bounds__(XF_CTA) xe_few_grad_kernel(const XfArgs a)
{
    const int i = blockIdx.x * (XF_CTA / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (i >= a.rows) return;
    const int own = xf_own(a, i);
    float g[2] = {};
    if (own >= 0) {
        const xf_row<T> row(a, i);
        const float2 st = a.stats[i];
        const float w = a.weight ? a.weight[i] : 1.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j = lane + 32 * h;
            g[h] = j >= a.vocab ? 0.0f : w * (j == own ? st.y : expf(row.z[h] - st.x));
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (lane + 32 * h < a.vocab) a.g[(int64_t)i * a.vocab + lane + 32 * h] = g[h];
    if (!a.dx) return;
    float d[XF_PER] = {};
    if (own >= 0)
        for (int j = 0; j < a.vocab; ++j) {
            const float f = __shfl_sync(0xffffffffu, j < 32 ? g[0] : g[1], j & 31);
            const T* const w = static_cast<const T*>(a.W) + j * a.ldw;
#pragma unroll
            for (int u = 0; u < XF_PER; ++u)
                if (lane + 32 * u < a.k) d[u] = fmaf(f, to_f32(w[lane + 32 * u]), d[u]);
        }
    T* const to = static_cast<T*>(a.dx) + i * a.lddx;
#pragma unroll
    for (int u = 0; u < XF_PER; ++u)
        if (lane + 32 * u < a.k) to[lane + 32 * u] = from_f32<T>(d[u]);
}

// dW: 32 columns and 4 classes a CTA, 16 threads' shares of the rows
template <typename T> __global__ void __launch_bounds__(512) xe_few_weight_kernel(const XfArgs a)
{
    __shared__ float of[16][4][32];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, col = blockIdx.x * 32 + lane, j0 = blockIdx.y * 4;
    float t[4] = {};
#pragma unroll 4
    for (int i = g; i < a.rows; i += 16) {
        const bool counts = xf_own(a, i) >= 0;   // (a row that is left out may hold anything)
        const float x = counts && col < a.k ? to_f32(static_cast<const T*>(a.x)[i * a.ldx + col]) : 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) t[c] = fmaf(a.g[(int64_t)i * a.vocab + min(j0 + c, a.vocab - 1)], x, t[c]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) of[g][c][lane] = t[c];
    __syncthreads();
    if (g >= 4 || col >= a.k || j0 + g >= a.vocab) return;
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) s += of[r][g][lane];
    static_cast<T*>(a.dW)[(j0 + g) * a.lddw + col] = from_f32<T>(s);
}

}  // namespace

bool xe_few_takes(int64_t rows, int64_t vocab, int64_t k) { return rows <= XF_ROWS && vocab <= XF_CLASSES && k <= XF_COLS; }
size_t xe_few_bytes(int64_t rows, int64_t vocab) { return (size_t)rows * vocab * sizeof(float); }

int xe_few_loss(s2v_ctx* ctx, cudaStream_t st, int64_t rows, int64_t vocab, int64_t k, int type, const void* x, int64_t ldx, const void* W, int64_t ldw, const int32_t* target,
                const float* row_weight, float* loss, float* stats)
{
    const XfArgs a{(int)rows, (int)vocab, (int)k, ldx, ldw, 0, 0, x, W, target, row_weight, loss, reinterpret_cast<float2*>(stats), nullptr, nullptr, nullptr};
    return s2v_by_dtype(type, [&](auto t) {
        xe_few_loss_kernel<decltype(t)><<<(unsigned)((rows + XF_CTA / 32 - 1) / (XF_CTA / 32)), XF_CTA, 0, st>>>(a);
        S2V_CHECK_LAUNCH(ctx, "xe_few_loss_kernel");
        return (int)S2V_OK;
    });
}

int xe_few_grad(s2v_ctx* ctx, cudaStream_t st, int64_t rows, int64_t vocab, int64_t k, int type, const void* x, int64_t ldx, const void* W, int64_t ldw, const int32_t* target,
                const float* row_weight, const float* stats, void* workspace, void* dx, int64_t lddx, void* dW, int64_t lddw)
{
    const XfArgs a{(int)rows, (int)vocab, (int)k, ldx, ldw, lddx, lddw, x, W, target, row_weight, nullptr, reinterpret_cast<float2*>(const_cast<float*>(stats)), static_cast<float*>(workspace), dx, dW};
    return s2v_by_dtype(type, [&](auto t) {
        using T = decltype(t);
        xe_few_grad_kernel<T><<<(unsigned)((rows + XF_CTA / 32 - 1) / (XF_CTA / 32)), XF_CTA, 0, st>>>(a);
        S2V_CHECK_LAUNCH(ctx, "xe_few_grad_kernel");
        if (dW) {
            xe_few_weight_kernel<T><<<dim3((unsigned)((k + 31) / 32), (unsigned)((vocab + 3) / 4)), 512, 0, st>>>(a);
            S2V_CHECK_LAUNCH(ctx, "xe_few_weight_kernel");
        }
        return (int)S2V_OK;
    });
}
