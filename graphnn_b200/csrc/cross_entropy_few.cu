// Softmax cross entropy of z = x W^T and its gradients for up to 64 classes, 512 columns and 512 rows: fp32 arithmetic, one launch for the loss and two for the gradients.
// A CTA has a row of x in shared memory; its warps share the classes, a logit being a sum over the lanes, and its threads the columns of dx.  What bounds it is the
// latency of a chain of steps (a warp a row, 35 classes one after the other: 3 x 35 x 449 fp16, a step, 158 us).
#include "cross_entropy_few.cuh"
#include "cross_entropy_rows.cuh"

namespace
{

constexpr int XF_CLASSES = 64, XF_COLS = 512, XF_ROWS = 512, XF_CTA = 256, XF_WARPS = XF_CTA / 32;

struct XfArgs {
    int rows, vocab, k;
    int64_t ldx, ldw, lddx, lddw;
    const void* x;
    const void* W;
    xe_rows of;
    float* loss;
    float2* stats;
    float* g;   // [rows][vocab]
    void* dx;
    void* dW;
};

// row i's logits to z[64], by the whole CTA
template <typename T> __device__ __forceinline__ void xf_logits(const XfArgs& a, int i, float* x, float* z)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int c = threadIdx.x; c < a.k; c += XF_CTA) x[c] = to_f32(static_cast<const T*>(a.x)[i * a.ldx + c]);
    __syncthreads();
    constexpr int AT_ONCE = 4;   // classes of a warp
    for (int j0 = warp; j0 < a.vocab; j0 += AT_ONCE * XF_WARPS) {
        float s[AT_ONCE] = {};
#pragma unroll 4
        for (int c = lane; c < a.k; c += 32) {
            const float v = x[c];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) s[u] = fmaf(v, to_f32(static_cast<const T*>(a.W)[min(j0 + u * XF_WARPS, a.vocab - 1) * a.ldw + c]), s[u]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1)
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], o);
        if (lane == 0) {
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u)
                if (j0 + u * XF_WARPS < a.vocab) z[j0 + u * XF_WARPS] = s[u];
        }
    }
    __syncthreads();
}

template <typename T> __global__ void __launch_bounds__(XF_CTA) xe_few_loss_kernel(const XfArgs a)
{
    __shared__ float x[XF_COLS], z[XF_CLASSES];
    const int i = blockIdx.x, own = (int)(a.stats ? a.of.its(i) : a.of.own(i));
    if (own < 0) {
        if (threadIdx.x == 0) {
            a.loss[i] = 0.0f;
            if (a.stats) a.stats[i] = make_float2(0.0f, 0.0f);
        }
        return;
    }
    xf_logits<T>(a, i, x, z);
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    const float mine = z[own];
    // the other classes' exponentials, relative to the largest of them
    float top = -INFINITY;
#pragma unroll
    for (int j = lane; j < XF_CLASSES; j += 32)
        if (j < a.vocab && j != own) top = fmaxf(top, z[j]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float from = fabsf(top) == INFINITY ? 0.0f : top;
    float l = 0.0f;
#pragma unroll
    for (int j = lane; j < XF_CLASSES; j += 32)
        if (j < a.vocab && j != own) l += top == INFINITY ? NAN : expf(z[j] - from);
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) xe_finish(a.of, i, top, l, mine, a.loss, a.stats);
}

// G and dx
template <typename T> __global__ void __launch_bounds__(XF_CTA) xe_few_grad_kernel(const XfArgs a)
{
    __shared__ float x[XF_COLS], z[XF_CLASSES];
    const int i = blockIdx.x, own = (int)a.of.own(i);
    if (own >= 0) {
        xf_logits<T>(a, i, x, z);
        if (threadIdx.x < a.vocab) {
            const float2 st = a.stats[i];
            const int j = threadIdx.x;
            const float g = (a.of.weight ? a.of.weight[i] : 1.0f) * (j == own ? st.y : expf(z[j] - st.x));
            z[j] = g, a.g[(int64_t)i * a.vocab + j] = g;
        }
        __syncthreads();
    } else if (threadIdx.x < a.vocab) a.g[(int64_t)i * a.vocab + threadIdx.x] = 0.0f;
    if (!a.dx) return;
    for (int c = threadIdx.x; c < a.k; c += XF_CTA) {
        float d = 0.0f;
        if (own >= 0) {
#pragma unroll 8
            for (int j = 0; j < a.vocab; ++j) d = fmaf(z[j], to_f32(static_cast<const T*>(a.W)[j * a.ldw + c]), d);
        }
        static_cast<T*>(a.dx)[i * a.lddx + c] = from_f32<T>(d);
    }
}

// dW: 32 columns and 4 classes a CTA, 16 threads' shares of the rows
template <typename T> __global__ void __launch_bounds__(512) xe_few_weight_kernel(const XfArgs a)
{
    __shared__ float of[16][4][32];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, col = blockIdx.x * 32 + lane, j0 = blockIdx.y * 4;
    float t[4] = {};
#pragma unroll 4
    for (int i = g; i < a.rows; i += 16) {
        const bool counts = a.of.own(i) >= 0;   // (a row that is left out may hold anything)
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
    const XfArgs a{(int)rows, (int)vocab, (int)k, ldx, ldw, 0, 0, x, W, {target, row_weight, vocab}, loss, reinterpret_cast<float2*>(stats), nullptr, nullptr, nullptr};
    return s2v_by_dtype(type, [&](auto t) {
        xe_few_loss_kernel<decltype(t)><<<(unsigned)rows, XF_CTA, 0, st>>>(a);
        S2V_CHECK_LAUNCH(ctx, "xe_few_loss_kernel");
        return (int)S2V_OK;
    });
}

int xe_few_grad(s2v_ctx* ctx, cudaStream_t st, int64_t rows, int64_t vocab, int64_t k, int type, const void* x, int64_t ldx, const void* W, int64_t ldw, const int32_t* target,
                const float* row_weight, const float* stats, void* workspace, void* dx, int64_t lddx, void* dW, int64_t lddw)
{
    const XfArgs a{(int)rows, (int)vocab, (int)k, ldx, ldw, lddx, lddw, x, W, {target, row_weight, vocab}, nullptr, reinterpret_cast<float2*>(const_cast<float*>(stats)), static_cast<float*>(workspace), dx, dW};
    return s2v_by_dtype(type, [&](auto t) {
        using T = decltype(t);
        xe_few_grad_kernel<T><<<(unsigned)rows, XF_CTA, 0, st>>>(a);
        S2V_CHECK_LAUNCH(ctx, "xe_few_grad_kernel");
        if (dW) {
            xe_few_weight_kernel<T><<<dim3((unsigned)((k + 31) / 32), (unsigned)((vocab + 3) / 4)), 512, 0, st>>>(a);
            S2V_CHECK_LAUNCH(ctx, "xe_few_weight_kernel");
        }
        return (int)S2V_OK;
    });
}
