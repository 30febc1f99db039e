// Distillation: Kullback-Leibler loss of a student's logits against a teacher's top logits, and its gradient.
//
// The listed columns and all others are summed apart, each relative to its own largest z: S_in = sum of exp((z - M_in) / T) over the list,
// S_out the same over the rest.  With M the larger maximum and total = S_in exp((M_in - M) / T) + S_out exp((M_out - M) / T),
//     log q_j = (z_j - M) / T - log total,     log s = -log(1 + exp(d)),  d = log(S_in / S_out) + (M_in - M_out) / T.
// Taking one sum from the other's total would lose s (or 1 - s) where the student gives nearly everything (or nothing) to the list, and one
// maximum for both would lose the smaller sum where they are far apart (logits masked with the type's lowest value).  Whatever exists once per
// row or per entry is computed in 64 bits, the sums over columns in fp32.
#include "elem_types.cuh"

namespace
{

constexpr int DT_TOP = 256;            // most entries of a list
constexpr int DT_THREADS = 256;        // at least DT_TOP: a thread per entry
constexpr int64_t DT_COLS = 1 << 20;   // a bit per column in shared memory
constexpr int DT_SITE = 7;             // status word: a class outside the row

struct DtArgs {
    int64_t rows, cols, ldz, ldt, lddz;
    const void* z;
    const int32_t* idx;
    const void* t;
    const float* t_lse;
    const float* row_weight;
    float* loss;
    float* stats;
    void* dz;
    s2v_device_status* status;
    float temperature;
    int top, t_type;
};

struct DtShared {
    double sum[8];
    float zk[DT_TOP], mx[8], sm[8];
    double p[DT_TOP];
    int idx[DT_TOP];   // -1: no entry
    int any;
};

__device__ __forceinline__ float dt_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float dt_finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }   // so that a difference from it is no NaN

__device__ __forceinline__ double dt_block_sum(double v, DtShared& s)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) s.sum[warp] = v;
    __syncthreads();
    double r = 0.0;
    for (int w = 0; w < DT_THREADS / 32; ++w) r += s.sum[w];
    return r;
}
__device__ __forceinline__ float dt_block_max(float v, DtShared& s)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) s.mx[warp] = v;
    __syncthreads();
    float r = s.mx[0];
    for (int w = 1; w < DT_THREADS / 32; ++w) r = fmaxf(r, s.mx[w]);
    return r;
}

// what follows from a row's two sums
struct DtRow {
    double M, out, total, log_s;   // out: exp((M_out - M) / T)
    __device__ __forceinline__ DtRow(float m_in, double s_in, float m_out, double s_out, float temperature)
    {
        M = (double)fmaxf(m_in, m_out);
        out = s_out == 0.0 ? 0.0 : exp(((double)m_out - M) / temperature);
        total = M == -INFINITY ? NAN : (s_in == 0.0 ? 0.0 : s_in * exp(((double)m_in - M) / temperature)) + s_out * out;
        const double d = s_in == 0.0 ? -INFINITY : log(s_in / s_out) + ((double)m_in - (double)m_out) / temperature;
        log_s = d > 0.0 ? -d - log1p(exp(-d)) : -log1p(exp(d));
    }
};

// A CTA per row.
template <typename T, bool GRAD_ONLY>
__global__ void __launch_bounds__(DT_THREADS) distill_rows_kernel(const DtArgs a)
{
    extern __shared__ uint32_t listed[];   // a bit per column: whether an entry names it
    __shared__ DtShared s;
    const int tid = threadIdx.x;
    const float c = 1.4426950408889634f / a.temperature;
    for (int64_t w = tid; w < (a.cols + 31) / 32; w += DT_THREADS) listed[w] = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* const z = static_cast<const T*>(a.z) + r * a.ldz;
        T* const dz = a.dz ? static_cast<T*>(a.dz) + r * a.lddz : nullptr;
        const float weight = a.row_weight ? a.row_weight[r] : 1.0f;
        // the list: entries, p, their sum
        int id = -1;
        float tv = -INFINITY;
        if (tid < a.top) {
            id = a.idx[r * a.ldt + tid];
            if (id >= a.cols) {
                a.status->code = S2V_ERR_INVALID_ARG;
                a.status->where = DT_SITE;
                id = -1;
            }
            const int64_t at = r * a.ldt + tid;
            if (id >= 0)
                tv = a.t_type == S2V_F32 ? static_cast<const float*>(a.t)[at] : a.t_type == S2V_F16 ? to_f32(static_cast<const __half*>(a.t)[at])
                                                                                                   : to_f32(static_cast<const __nv_bfloat16*>(a.t)[at]);
        }
        const bool some = __syncthreads_or(id >= 0);
        const float tmax = dt_block_max(tv, s);
        double p = 0.0, given, rest = 0.0;
        if (a.t_lse) {
            if (id >= 0) p = exp((double)tv / a.temperature - (double)a.t_lse[r]);
            given = dt_block_sum(p, s);
            rest = given > 1.0 ? 0.0 : 1.0 - given;
        } else {
            if (id >= 0) p = exp(((double)tv - (double)dt_finite_or_zero(tmax)) / a.temperature);
            const double total = dt_block_sum(p, s);
            p /= total;
            given = total - total + 1.0;   // one, and NaN where the list holds NaN or +infinity
        }
        const bool skip = !some || (!a.t_lse && tmax == -INFINITY);
        if (skip || (weight == 0.0f && !a.stats) || (GRAD_ONLY && weight == 0.0f)) {   // (the same for the whole CTA)
            if (!GRAD_ONLY && tid == 0) a.loss[r] = 0.0f;
            if (!GRAD_ONLY && a.stats && tid < 4) a.stats[4 * r + tid] = 0.0f;
            if (dz)
                for (int64_t j = tid; j < a.cols; j += DT_THREADS) dz[j] = from_f32<T>(0.0f);
            __syncthreads();
            continue;
        }
        __syncthreads();
        if (tid < a.top) {
            s.idx[tid] = id;
            s.p[tid] = p;
            if (id >= 0) atomicOr(&listed[id >> 5], 1u << (id & 31));
        }
        const float zk = id >= 0 ? to_f32(z[id]) : -INFINITY;
        __syncthreads();
        // the first entry of a column stands for it; p of all its entries
        bool first = id >= 0;
        double p_all = 0.0;
        if (id >= 0)
            for (int k = 0; k < a.top; ++k)
                if (s.idx[k] == id) {
                    p_all += s.p[k];
                    if (k < tid) first = false;
                }
        float m_in, m_out;
        double s_in, s_out;
        if constexpr (GRAD_ONLY) {
            m_out = a.stats[4 * r], s_out = (double)a.stats[4 * r + 1];
            m_in = a.stats[4 * r + 2], s_in = (double)a.stats[4 * r + 3];
        } else {
            float m = -INFINITY, sum = 0.0f;
            for (int64_t j = tid; j < a.cols; j += DT_THREADS) {
                if (listed[j >> 5] >> (j & 31) & 1) continue;
                const float v = to_f32(z[j]);
                if (v > m) {
                    sum *= dt_exp2((m - v) * c);   // (m = -infinity: no sum yet)
                    m = v;
                }
                sum += dt_exp2((v - dt_finite_or_zero(m)) * c);
            }
            m_out = dt_block_max(m, s);
            s_out = dt_block_sum((double)(sum * dt_exp2((m - dt_finite_or_zero(m_out)) * c)), s);
            m_in = dt_block_max(zk, s);
            s_in = dt_block_sum(first ? exp(((double)zk - (double)dt_finite_or_zero(m_in)) / a.temperature) : 0.0, s);
        }
        const DtRow row(m_in, s_in, m_out, s_out, a.temperature);
        if constexpr (!GRAD_ONLY) {
            double kl = 0.0;
            if (id >= 0 && p != 0.0) kl = p * (log(p) - (((double)zk - row.M) / a.temperature - log(row.total)));
            kl = dt_block_sum(kl, s);
            if (rest != 0.0) {
                if (s_out != 0.0) kl += rest * (log1p(-given) - row.log_s);
                else if (rest > 1.0 / 65536.0) kl = INFINITY;
            }
            if (!(row.total > 0.0)) kl = NAN;
            if (tid == 0) {
                a.loss[r] = weight == 0.0f ? 0.0f : (float)(kl * weight);
                if (a.stats) *reinterpret_cast<float4*>(a.stats + 4 * r) = make_float4(m_out, (float)s_out, m_in, (float)s_in);
            }
        }
        if (dz) {
            const double scale = (double)weight / a.temperature;
            const float out = weight == 0.0f ? 0.0f : !(row.total > 0.0) ? NAN : s_out == 0.0 ? 0.0f : (float)(scale * ((given + rest) * row.out / row.total - rest / s_out));
            const float base = dt_finite_or_zero(m_out);
            __syncthreads();   // every listed z has been read
            for (int64_t j = tid; j < a.cols; j += DT_THREADS) {
                if (listed[j >> 5] >> (j & 31) & 1) continue;
                dz[j] = from_f32<T>(out == 0.0f ? 0.0f : dt_exp2((to_f32(z[j]) - base) * c) * out);
            }
            if (first) dz[id] = from_f32<T>(weight == 0.0f ? 0.0f : (float)(scale * ((given + rest) * exp(((double)zk - row.M) / a.temperature) / row.total - p_all)));
        }
        __syncthreads();
        if (id >= 0) listed[id >> 5] = 0;   // (a word, by all its entries)
        __syncthreads();
    }
}

int dt_launch(s2v_ctx* ctx, s2v_stream stream, int z_type, bool grad_only, const DtArgs& a)
{
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    const size_t bits = (size_t)((a.cols + 31) / 32) * 4;
    const int64_t cap = (int64_t)ctx->sm_count * 8;
    const unsigned grid = (unsigned)(a.rows < cap ? a.rows : cap);
    return s2v_by_dtype(z_type, [&](auto type) {
        using T = decltype(type);
        if (grad_only) {
            S2V_CUDA_OK(ctx, s2v_allow_shared(distill_rows_kernel<T, true>, DT_COLS / 8));
            distill_rows_kernel<T, true><<<grid, DT_THREADS, bits, st>>>(a);
        } else {
            S2V_CUDA_OK(ctx, s2v_allow_shared(distill_rows_kernel<T, false>, DT_COLS / 8));
            distill_rows_kernel<T, false><<<grid, DT_THREADS, bits, st>>>(a);
        }
        S2V_CHECK_LAUNCH(ctx, "distill_rows_kernel");
        return (int)S2V_OK;
    });
}

int dt_check(s2v_ctx* ctx, const char* name, int z_type, const DtArgs& a)
{
    const std::string who(name);
    if (a.rows < 0 || a.cols <= 0 || a.top <= 0) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": negative or empty size");
    if (!s2v_dtype_ok(z_type) || !s2v_dtype_ok(a.t_type)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": unknown element type");
    if (!(a.temperature >= 1e-30f && a.temperature <= 1e30f)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": temperature outside [1e-30, 1e30]");
    if (a.rows == 0) return S2V_OK;
    if (!a.z || !a.idx || !a.t) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": NULL pointer");
    if (a.top > DT_TOP) return s2v_fail(ctx, S2V_ERR_UNSUPPORTED, who + ": more than 256 entries a row");
    if (a.cols > DT_COLS) return s2v_fail(ctx, S2V_ERR_UNSUPPORTED, who + ": more than 1,048,576 columns");
    if (a.rows > 1 && (a.ldz < a.cols || a.ldt < a.top || (a.dz && a.lddz < a.cols)))
        return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": leading dimension below the number of columns");
    const size_t es = s2v_dtype_bytes(z_type);
    if (reinterpret_cast<uintptr_t>(a.z) % es || reinterpret_cast<uintptr_t>(a.dz) % es || reinterpret_cast<uintptr_t>(a.t) % s2v_dtype_bytes(a.t_type))
        return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": misaligned pointer");
    if (!s2v_aligned16(a.stats)) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": stats must be 16-byte aligned");
    if (a.dz == a.z && a.rows > 1 && a.lddz != a.ldz) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, who + ": dz in the place of z needs the same leading dimension");
    return S2V_OK;
}

}  // namespace

extern "C" {

int s2v_distill_topk(s2v_ctx* ctx, s2v_stream stream, int64_t rows, int64_t cols, int z_type, const void* z, int64_t ldz, int top, const int32_t* idx,
                     int t_type, const void* t, int64_t ldt, const float* t_lse, float temperature, const float* row_weight, float* loss, float* stats,
                     void* dz, int64_t lddz)
{
    S2V_ENTER(ctx);
    const DtArgs a{rows, cols, ldz, ldt, lddz, z, idx, t, t_lse, row_weight, loss, stats, dz, ctx->dstatus_dev, temperature, top, t_type};
    const int rc = dt_check(ctx, "distill_topk", z_type, a);
    if (rc != S2V_OK || rows == 0) return rc;
    if (!loss) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "distill_topk: NULL loss");
    return dt_launch(ctx, stream, z_type, false, a);
}

int s2v_distill_topk_grad(s2v_ctx* ctx, s2v_stream stream, int64_t rows, int64_t cols, int z_type, const void* z, int64_t ldz, int top, const int32_t* idx,
                          int t_type, const void* t, int64_t ldt, const float* t_lse, float temperature, const float* row_weight, const float* stats,
                          void* dz, int64_t lddz)
{
    S2V_ENTER(ctx);
    const DtArgs a{rows, cols, ldz, ldt, lddz, z, idx, t, t_lse, row_weight, nullptr, const_cast<float*>(stats), dz, ctx->dstatus_dev, temperature, top, t_type};
    const int rc = dt_check(ctx, "distill_topk_grad", z_type, a);
    if (rc != S2V_OK || rows == 0) return rc;
    if (!stats || !dz) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "distill_topk_grad: NULL pointer");
    return dt_launch(ctx, stream, z_type, true, a);
}

}  // extern "C"
