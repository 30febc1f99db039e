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
constexpr int64_t DT_COLS = 1 << 20;   // most columns
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

__device__ __forceinline__ float dt_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float dt_finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }   // so that a difference from it is no NaN

template <typename V> __device__ __forceinline__ V dt_warp_sum(V v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float dt_warp_max(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// ---------------------------------------------------------------- sums and gradients of pieces of 16 bytes
// e[i] = exp2((x[i] + minus_m) * c), two at a time
template <int N> __device__ __forceinline__ void dt_exps(const float* x, float minus_m, float c, float* e)
{
    if constexpr (N == 1) {
        e[0] = dt_exp2((x[0] + minus_m) * c);
    } else {
        uint64_t m2, c2;
        asm("mov.b64 %0, {%1, %1};" : "=l"(m2) : "f"(minus_m));
        asm("mov.b64 %0, {%1, %1};" : "=l"(c2) : "f"(c));
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            uint64_t v;
            asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x[i]), "f"(x[i + 1]));
            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(m2));
            asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(c2));
            asm("mov.b64 {%0, %1}, %2;" : "=f"(e[i]), "=f"(e[i + 1]) : "l"(v));
            e[i] = dt_exp2(e[i]);
            e[i + 1] = dt_exp2(e[i + 1]);
        }
    }
}

struct DtSum {   // of exp((z - m) / T), relative to the largest z
    float m, s;
    // (x is overwritten where columns are listed: few pieces have any)
    template <int N> __device__ __forceinline__ void add(float* x, uint32_t listed, float c)
    {
        if (listed) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (listed >> e & 1) x[e] = -INFINITY;
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < N; ++e) top = fmaxf(top, x[e]);
        if (top > m) {
            s *= dt_exp2((m - top) * c);   // (m = -infinity: no sum yet)
            m = top;
        }
        float e[N];
        dt_exps<N>(x, -dt_finite_or_zero(m), c, e);
#pragma unroll
        for (int w = N / 2; w; w >>= 1)
#pragma unroll
            for (int i = 0; i < w; ++i) e[i] += e[i + w];
        s += e[0];
    }
    __device__ __forceinline__ void join_warp(float c)
    {
        const float top = dt_warp_max(m);
        s = dt_warp_sum(s * dt_exp2((m - dt_finite_or_zero(top)) * c));
        m = top;
    }
};

// zeros in the columns of a row that falls to this thread, one of `threads`
template <typename T> __device__ __forceinline__ void dt_zero_row(T* dz, int64_t cols, int at, int threads)
{
    const row_pieces<T> row(dz, cols);
    if (at < row.head) dz[at] = from_f32<T>(0.0f);
    if (at < row.tail) dz[cols - 1 - at] = from_f32<T>(0.0f);
    uint4* const to = reinterpret_cast<uint4*>(dz + row.head);
    for (int p = at; p < row.pieces; p += threads) to[p] = make_uint4(0, 0, 0, 0);
}

// gradient of a piece; listed columns are written by their entries
template <typename T> __device__ __forceinline__ void dt_store(T* to, bool whole, const uint4& v, uint32_t listed, float base, float outer, float c)
{
    constexpr int N = PIECE<T>;
    float x[N], e[N];
    unpack_piece(v, x, T());
    dt_exps<N>(x, -base, c, e);
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] *= outer;
    if (whole && listed == 0) {
        __stcs(reinterpret_cast<uint4*>(to), pack_piece(e, T()));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!(listed >> i & 1)) to[i] = from_f32<T>(e[i]);
    }
}

// ---------------------------------------------------------------- the list
// What a row's list adds up to, over any part of its entries; P_k = exp((t_k - t_max) / T), or exp(t_k / T - t_lse) where that is given:
//     Z = sum P,  A = sum P log P,  B = sum P (z_idx - m) / T,  s = sum of exp((z_idx - m) / T) over the columns,  m = the largest z_idx
struct DtList {
    double Z, A, B, s;
    float m;
};
__device__ __forceinline__ int dt_load_id(const DtArgs& a, int64_t r, int k)
{
    const int id = k < a.top ? __ldg(a.idx + r * a.ldt + k) : -1;
    if (id < a.cols) return id < 0 ? -1 : id;
    a.status->code = S2V_ERR_INVALID_ARG;
    a.status->where = DT_SITE;
    return -1;
}
__device__ __forceinline__ float dt_load_t(const DtArgs& a, int64_t r, int k)
{
    const int64_t at = r * a.ldt + k;
    return a.t_type == S2V_F32 ? __ldg(static_cast<const float*>(a.t) + at) : a.t_type == S2V_F16 ? to_f32(static_cast<const __half*>(a.t)[at])
                                                                                                   : to_f32(static_cast<const __nv_bfloat16*>(a.t)[at]);
}
// log P of an entry
__device__ __forceinline__ double dt_log_p(const DtArgs& a, float tv, float tmax, double t_lse, double inv_t)
{
    return a.t_lse ? (double)tv * inv_t - t_lse : ((double)tv - (double)dt_finite_or_zero(tmax)) * inv_t;
}

// an entry's part of Z, A and B (B relative to l.m, the largest listed z)
__device__ __forceinline__ void dt_count(const DtArgs& a, DtList& l, float tv, float tmax, double t_lse, float zk, double inv_t)
{
    const double lp = dt_log_p(a, tv, tmax, t_lse, inv_t), P = exp(lp);
    l.Z += P;
    if (P != 0.0) {
        l.A += P * lp;
        l.B += P * (((double)zk - (double)dt_finite_or_zero(l.m)) * inv_t);
    }
}

// ---------------------------------------------------------------- a row, once its sums are known
struct DtCoef {
    float M;            // the larger maximum (0 where there is none)
    float p_scale;      // p = P * p_scale
    float inner;        // a listed column's gradient: inner * exp((z - M) / T) - scale * p
    float outer;        // any other's: outer * exp((z - m_out) / T)
    float scale;        // row_weight / T
};
__device__ __forceinline__ DtCoef dt_coefficients(const DtArgs& a, double Z, const DtSum& in, const DtSum& out, float weight, float c)
{
    DtCoef k;
    const float m = fmaxf(in.m, out.m);
    k.M = dt_finite_or_zero(m);
    const float e_out = out.s == 0.0f ? 0.0f : dt_exp2((out.m - k.M) * c), e_in = in.s == 0.0f ? 0.0f : dt_exp2((in.m - k.M) * c);
    const float total = m == -INFINITY ? NAN : in.s * e_in + out.s * e_out;
    float given, rest;
    if (a.t_lse) {
        given = (float)Z;
        rest = Z > 1.0 ? 0.0f : (float)(1.0 - Z);
        k.p_scale = 1.0f;
    } else {
        given = (float)(Z - Z + 1.0);   // one, and NaN where the list holds NaN or +infinity
        rest = 0.0f;
        k.p_scale = 1.0f / (float)Z;
    }
    k.scale = weight / a.temperature;
    const float both = (given + rest) / total;
    k.inner = k.scale * both;
    k.outer = k.scale * (out.s == 0.0f && total == total ? 0.0f : both * e_out - rest / out.s);
    return k;
}
__device__ __forceinline__ float dt_loss(const DtArgs& a, const DtList& l, float m_out, double s_out, float weight, double inv_t)
{
    const float mf = fmaxf(l.m, m_out);
    if (mf == -INFINITY) return NAN;
    const double M = (double)mf;
    const double total = (l.s == 0.0 ? 0.0 : l.s * exp(((double)l.m - M) * inv_t)) + (s_out == 0.0 ? 0.0 : s_out * exp(((double)m_out - M) * inv_t));
    const double lse = log(total);   // above M / T
    // sum of p (log p - log q), log q = (z - M) / T - lse; B is relative to l.m
    const double from = l.m == -INFINITY ? 0.0 : ((double)l.m - M) * inv_t;
    double kl, rest = 0.0;
    if (a.t_lse) {
        kl = l.A - (l.B + l.Z * from) + l.Z * lse;
        rest = l.Z > 1.0 ? 0.0 : 1.0 - l.Z;
    } else {
        kl = (l.A - (l.B + l.Z * from)) / l.Z - log(l.Z) + lse;
    }
    if (rest != 0.0) {
        if (s_out != 0.0) {
            const double d = l.s == 0.0 ? -INFINITY : log(l.s / s_out) + ((double)l.m - (double)m_out) * inv_t;
            kl += rest * (log1p(-l.Z) + (d > 0.0 ? d + log1p(exp(-d)) : log1p(exp(d))));
        } else if (rest > 1.0 / 65536.0) {
            kl = INFINITY;
        }
    }
    return (float)(kl * weight);
}

// ---------------------------------------------------------------- rows of up to 256 pieces: a warp each
// The row stays in registers between the sums and the gradient.
constexpr int DW_WARPS = 4, DW_PIECES = 8;   // pieces a lane
struct DwShared {
    double P[DT_TOP];
    float z[DT_TOP];
    int id[DT_TOP];
    uint32_t mask[(DW_PIECES * 32 + 4 + 31) / 32 * 8 + 1];   // a byte per piece, then one for the head and one for the tail
};

template <typename T, int NV, bool GRAD_ONLY>
__global__ void __launch_bounds__(32 * DW_WARPS) distill_warp_kernel(const DtArgs a)
{
    __shared__ DwShared shared[DW_WARPS];
    DwShared& s = shared[threadIdx.x >> 5];
    constexpr int N = PIECE<T>, EDGE = DW_PIECES * 32;   // mask bytes of the head and the tail: EDGE, EDGE + 1
    const int lane = threadIdx.x & 31;
    const double inv = 1.0 / (double)a.temperature;
    const float inv_t = 1.0f / a.temperature, c = 1.4426950408889634f / a.temperature;
    const uint8_t* const mask = reinterpret_cast<const uint8_t*>(s.mask);
    for (int w = lane; w < (int)(sizeof(s.mask) / 4); w += 32) s.mask[w] = 0;
    __syncwarp();
    const int64_t step = (int64_t)gridDim.x * DW_WARPS;
    for (int64_t r = (int64_t)blockIdx.x * DW_WARPS + (threadIdx.x >> 5); r < a.rows; r += step) {
        const T* const z = static_cast<const T*>(a.z) + r * a.ldz;
        T* const dz = a.dz ? static_cast<T*>(a.dz) + r * a.lddz : nullptr;
        const float weight = a.row_weight ? __ldg(a.row_weight + r) : 1.0f;
        const row_pieces<T> row(z, a.cols);
        float tmax = -INFINITY;
        bool some = false;
        for (int k = lane; k < a.top; k += 32) {
            const int id = dt_load_id(a, r, k);
            s.id[k] = id;
            if (id < 0) continue;
            some = true;
            tmax = fmaxf(tmax, dt_load_t(a, r, k));
        }
        some = __any_sync(0xffffffffu, some);
        tmax = dt_warp_max(tmax);
        if (!some || (!a.t_lse && tmax == -INFINITY) || (weight == 0.0f && (GRAD_ONLY || !a.stats))) {
            if (!GRAD_ONLY && lane == 0) a.loss[r] = 0.0f;
            if (!GRAD_ONLY && a.stats && lane < 4) a.stats[4 * r + lane] = 0.0f;
            if (dz) dt_zero_row(dz, a.cols, lane, 32);
            __syncwarp();
            continue;
        }
        uint4 v[NV];
        const uint4* const zp = reinterpret_cast<const uint4*>(z + row.head);
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * 32 + lane < row.pieces) v[j] = zp[j * 32 + lane];
        // the scalar columns: the head's to the first lanes, the tail's to the last
        const bool in_head = lane < row.head, in_tail = lane >= 32 - row.tail;
        const int edge_at = in_head ? lane : (int)a.cols - 32 + lane, edge_bit = in_head ? lane : lane - (32 - row.tail);
        const float edge = in_head || in_tail ? to_f32(z[edge_at]) : -INFINITY;
        // the list
        const float t_lse = a.t_lse ? __ldg(a.t_lse + r) : 0.0f;
        DtList l{0.0, 0.0, 0.0, 0.0, -INFINITY};
        DtSum inner{-INFINITY, 0.0f};
        bool twice = false;
        for (int k = lane; k < a.top; k += 32) {
            const int id = s.id[k];
            if (id < 0) continue;
            const float zk = to_f32(z[id]);
            const double lp = dt_log_p(a, dt_load_t(a, r, k), tmax, (double)t_lse, inv), P = exp(lp);
            s.z[k] = zk, s.P[k] = P;
            l.Z += P;
            if (!GRAD_ONLY && P != 0.0) l.A += P * lp;
            inner.m = fmaxf(inner.m, zk);
            const int at = id - row.head, byte = at < 0 ? EDGE : at >= row.pieces * N ? EDGE + 1 : at / N, bit = at < 0 ? id : at >= row.pieces * N ? at - row.pieces * N : at % N;
            const uint32_t b = 1u << (8 * (byte & 3) + bit);
            twice |= (atomicOr(&s.mask[byte >> 2], b) & b) != 0;
        }
        twice = __any_sync(0xffffffffu, twice);
        __syncwarp();
        l.Z = dt_warp_sum(l.Z);
        inner.m = dt_warp_max(inner.m);
        const auto first = [&](int k, double* all) {   // whether entry k is the first of its column; P of all the column's entries
            *all = s.P[k];
            if (!twice) return true;
            bool f = true;
            double sum = 0.0;
            for (int i = 0; i < a.top; ++i)
                if (s.id[i] == s.id[k]) {
                    sum += s.P[i];
                    if (i < k) f = false;
                }
            *all = sum;
            return f;
        };
        DtSum outer{-INFINITY, 0.0f};
        const uint32_t edge_listed = in_head || in_tail ? mask[in_head ? EDGE : EDGE + 1] >> edge_bit & 1u : 1u;
        if constexpr (GRAD_ONLY) {
            const float4 st = __ldg(reinterpret_cast<const float4*>(a.stats) + r);
            outer = DtSum{st.x, st.y}, inner = DtSum{st.z, st.w};
        } else {
            for (int k = lane; k < a.top; k += 32) {
                if (s.id[k] < 0) continue;
                double all;
                const double x = ((double)s.z[k] - (double)dt_finite_or_zero(inner.m)) * inv;
                if (first(k, &all)) l.s += exp(x);
                if (s.P[k] != 0.0) l.B += s.P[k] * x;
            }
            l.A = dt_warp_sum(l.A), l.B = dt_warp_sum(l.B);
            l.s = dt_warp_sum(l.s);
            inner.s = (float)l.s, l.m = inner.m;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (j * 32 + lane < row.pieces) {
                    float x[N];
                    unpack_piece(v[j], x, T());
                    outer.template add<N>(x, mask[j * 32 + lane], c);
                }
            float edge_sum = edge;
            if (in_head || in_tail) outer.template add<1>(&edge_sum, edge_listed, c);
            outer.join_warp(c);
            if (a.stats && lane == 0) reinterpret_cast<float4*>(a.stats)[r] = make_float4(outer.m, outer.s, inner.m, inner.s);
            const float loss = dt_loss(a, l, outer.m, (double)outer.s, weight, inv);
            if (lane == 0) a.loss[r] = weight == 0.0f ? 0.0f : loss;
        }
        if (dz && weight == 0.0f) {   // (for the stats alone)
            __syncwarp();
            dt_zero_row(dz, a.cols, lane, 32);
        } else if (dz) {
            const DtCoef k = dt_coefficients(a, l.Z, inner, outer, weight, c);
            const float base = dt_finite_or_zero(outer.m);
            T* const dp = dz + row.head;
            const bool whole = (reinterpret_cast<uintptr_t>(dp) & 15) == 0;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (j * 32 + lane < row.pieces) dt_store(dp + (j * 32 + lane) * N, whole, v[j], mask[j * 32 + lane], base, k.outer, c);
            if (!edge_listed) dz[edge_at] = from_f32<T>(dt_exp2((edge - base) * c) * k.outer);
            for (int i = lane; i < a.top; i += 32) {
                double all;
                if (s.id[i] >= 0 && first(i, &all)) dz[s.id[i]] = from_f32<T>(k.inner * expf((s.z[i] - k.M) * inv_t) - k.scale * ((float)all * k.p_scale));
            }
        }
        __syncwarp();
        for (int k = lane; k < a.top; k += 32)
            if (s.id[k] >= 0) {
                const int at = s.id[k] - row.head, byte = at < 0 ? EDGE : at >= row.pieces * N ? EDGE + 1 : at / N;
                s.mask[byte >> 2] = 0;
            }
        __syncwarp();
    }
}

// ---------------------------------------------------------------- longer rows: a cluster of CTAs each
// Every CTA has an equal run of the row's pieces: the first NV of each thread stay in registers between the sums and the gradient, what a very
// long row has more is read again.  All CTAs take the list (a thread an entry) and count and write the listed columns of their own run, in fp32;
// the first CTA's first warp adds up the loss in 64 bits while the others write the gradient.
constexpr int DC_THREADS = 256, DC_WARPS = DC_THREADS / 32, DC_CTAS = 8;
static_assert(DC_THREADS == DT_TOP, "a thread an entry");
struct DcShared {
    float P[DT_TOP], t[DT_TOP], z[DT_TOP];
    int id[DT_TOP];
    float4 peer[2][DC_CTAS];            // outer and inner sums of the cluster's CTAs, two rows by turns
    float2 outer[DC_WARPS], inner[DC_WARPS];
    double Z[DC_WARPS];
    float tmax[DC_WARPS];
    uint32_t edge;                      // listed columns of the head (bits 0 to 7) and the tail (8 to 15)
};

template <typename T, int NV, bool GRAD_ONLY>
__global__ void __launch_bounds__(DC_THREADS, 3) distill_cluster_kernel(const DtArgs a, int ctas)
{
    extern __shared__ uint32_t dc_mask[];   // a byte per piece of this CTA
    __shared__ DcShared s;
    constexpr int N = PIECE<T>;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)(blockIdx.x % (unsigned)ctas);
    const double inv = 1.0 / (double)a.temperature;
    const float inv_t = 1.0f / a.temperature, c = 1.4426950408889634f / a.temperature;
    const uint8_t* const mask = reinterpret_cast<const uint8_t*>(dc_mask);
    const int most = (int)((a.cols / N + ctas - 1) / ctas);   // pieces of a CTA, at most
    for (int w = tid; w < (most + 3) / 4; w += DC_THREADS) dc_mask[w] = 0;
    if (tid == 0) s.edge = 0;
    int turn = 0;
    for (int64_t r = blockIdx.x / (unsigned)ctas; r < a.rows; r += gridDim.x / (unsigned)ctas) {
        const T* const z = static_cast<const T*>(a.z) + r * a.ldz;
        T* const dz = a.dz ? static_cast<T*>(a.dz) + r * a.lddz : nullptr;
        const float weight = a.row_weight ? __ldg(a.row_weight + r) : 1.0f, t_lse = a.t_lse ? __ldg(a.t_lse + r) : 0.0f;
        const int id = dt_load_id(a, r, tid);
        float tv = tid < a.top ? dt_load_t(a, r, tid) : -INFINITY;
        if (id < 0) tv = -INFINITY;
        const row_pieces<T> row(z, a.cols);
        const int first_piece = rank * most, pieces = max(0, min(most, row.pieces - first_piece));
        const uint4* const zp = reinterpret_cast<const uint4*>(z + row.head) + first_piece;
        const bool skip_weight = weight == 0.0f && (GRAD_ONLY || !a.stats);
        uint4 v[NV];
        if (!skip_weight) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (j * DC_THREADS + tid < pieces) v[j] = zp[j * DC_THREADS + tid];
        }
        {
            const float m = dt_warp_max(tv);
            if (lane == 0) s.tmax[warp] = m;
        }
        const bool some = __syncthreads_or(id >= 0);
        float tmax = s.tmax[0];
#pragma unroll
        for (int w = 1; w < DC_WARPS; ++w) tmax = fmaxf(tmax, s.tmax[w]);
        if (!some || (!a.t_lse && tmax == -INFINITY) || skip_weight) {   // (the same for all CTAs of the row)
            if (!GRAD_ONLY && rank == 0) {
                if (tid == 0) a.loss[r] = 0.0f;
                if (a.stats && tid < 4) a.stats[4 * r + tid] = 0.0f;
            }
            if (dz) dt_zero_row(dz, a.cols, rank * DC_THREADS + tid, ctas * DC_THREADS);
            __syncthreads();
            continue;
        }
        // the list: a thread an entry
        const int at = id - row.head, piece = at < 0 ? -1 : at / N - first_piece;   // (of this CTA's)
        const bool edge_entry = id >= 0 && (at < 0 || at >= row.pieces * N);
        const bool mine = edge_entry ? rank == (at < 0 ? 0 : ctas - 1) : id >= 0 && piece >= 0 && piece < pieces;
        uint32_t* const word = edge_entry ? &s.edge : &dc_mask[mine ? piece >> 2 : 0];
        const float zk = mine || (!GRAD_ONLY && rank == 0 && id >= 0) ? to_f32(z[id]) : -INFINITY;
        // (in 64 bits: what the list leaves to the others, 1 - Z, may be small)
        const double P = id >= 0 ? exp(dt_log_p(a, tv, tmax, (double)t_lse, inv)) : 0.0;
        bool twice = false;
        s.id[tid] = id;
        s.P[tid] = (float)P;
        s.t[tid] = tv;
        if (mine) {
            const uint32_t b = 1u << (!edge_entry ? 8 * (piece & 3) + at % N : at < 0 ? id : 8 + at - row.pieces * N);
            twice = (atomicOr(word, b) & b) != 0;
        }
        {
            const double Z = dt_warp_sum(P);
            if (lane == 0) s.Z[warp] = Z;
        }
        bool first = mine;   // the first entry of its column; P of all the column's entries
        float P_all = (float)P;
        if (__syncthreads_or(twice) && mine) {
            P_all = 0.0f;
            for (int k = 0; k < a.top; ++k)
                if (s.id[k] == id) {
                    P_all += s.P[k];
                    if (k < tid) first = false;
                }
        }
        // the scalar columns: the head's to the first CTA, the tail's to the last
        const bool in_head = rank == 0 && tid < row.head, in_tail = rank == ctas - 1 && tid >= 32 && tid < 32 + row.tail;
        const int edge_at = in_head ? tid : (int)a.cols - row.tail + tid - 32;
        const float edge = in_head || in_tail ? to_f32(z[edge_at]) : -INFINITY;
        const uint32_t edge_listed = in_head ? s.edge >> tid & 1u : in_tail ? s.edge >> (8 + tid - 32) & 1u : 1u;
        DtSum outer{-INFINITY, 0.0f}, inner{first ? zk : -INFINITY, first ? 1.0f : 0.0f};
        if constexpr (GRAD_ONLY) {
            const float4 st = __ldg(reinterpret_cast<const float4*>(a.stats) + r);
            outer = DtSum{st.x, st.y}, inner = DtSum{st.z, st.w};
        } else {
            // (a listed z of -infinity or NaN: 0 and NaN, as exp gives them)
            if (first && !(zk > -INFINITY)) inner.s = zk == -INFINITY ? 0.0f : NAN;
            if (zk == INFINITY && first) inner.s = NAN;
            s.z[tid] = zk;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (j * DC_THREADS + tid < pieces) {
                    float x[N];
                    unpack_piece(v[j], x, T());
                    outer.template add<N>(x, mask[j * DC_THREADS + tid], c);
                }
            for (int p = NV * DC_THREADS + tid; p < pieces; p += DC_THREADS) {
                float x[N];
                unpack_piece(zp[p], x, T());
                outer.template add<N>(x, mask[p], c);
            }
            float edge_sum = edge;
            if (in_head || in_tail) outer.template add<1>(&edge_sum, edge_listed, c);
            outer.join_warp(c);
            inner.join_warp(c);
            if (lane == 0) s.outer[warp] = make_float2(outer.m, outer.s), s.inner[warp] = make_float2(inner.m, inner.s);
            __syncthreads();
            // (every warp joins the warps' sums for itself)
            outer = lane < DC_WARPS ? DtSum{s.outer[lane].x, s.outer[lane].y} : DtSum{-INFINITY, 0.0f};
            inner = lane < DC_WARPS ? DtSum{s.inner[lane].x, s.inner[lane].y} : DtSum{-INFINITY, 0.0f};
            outer.join_warp(c);
            inner.join_warp(c);
            if (ctas > 1) {
                if (warp == 0 && lane < ctas) {
                    uint32_t to;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(&s.peer[turn][rank])), "r"(lane));
                    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(outer.m), "f"(outer.s), "f"(inner.m), "f"(inner.s) : "memory");
                }
                asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
                const float4 o = lane < ctas ? s.peer[turn][lane] : make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
                outer = DtSum{o.x, o.y}, inner = DtSum{o.z, o.w};
                outer.join_warp(c);
                inner.join_warp(c);
                turn ^= 1;
            }
            if (a.stats && rank == 0 && tid == DC_THREADS - 1) reinterpret_cast<float4*>(a.stats)[r] = make_float4(outer.m, outer.s, inner.m, inner.s);
        }
        if (dz && weight == 0.0f) {   // (for the stats alone; the cluster has read the row)
            if (ctas == 1) __syncthreads();
            dt_zero_row(dz, a.cols, rank * DC_THREADS + tid, ctas * DC_THREADS);
        } else if (dz) {
            const double Z = dt_warp_sum(lane < DC_WARPS ? s.Z[lane] : 0.0);
            const DtCoef k = dt_coefficients(a, Z, inner, outer, weight, c);
            const float base = dt_finite_or_zero(outer.m);
            T* const dp = dz + row.head + (int64_t)first_piece * N;
            const bool whole = (reinterpret_cast<uintptr_t>(dp) & 15) == 0;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (j * DC_THREADS + tid < pieces) dt_store(dp + (j * DC_THREADS + tid) * N, whole, v[j], mask[j * DC_THREADS + tid], base, k.outer, c);
            for (int p = NV * DC_THREADS + tid; p < pieces; p += DC_THREADS) dt_store(dp + (int64_t)p * N, whole, zp[p], mask[p], base, k.outer, c);
            if (!edge_listed) dz[edge_at] = from_f32<T>(dt_exp2((edge - base) * c) * k.outer);
            if (first) dz[id] = from_f32<T>(k.inner * expf((zk - k.M) * inv_t) - k.scale * (P_all * k.p_scale));
        }
        if (!GRAD_ONLY && rank == 0 && warp == 0) {
            DtList l{0.0, 0.0, 0.0, (double)inner.s, inner.m};
            for (int k = lane; k < a.top; k += 32)
                if (s.id[k] >= 0) dt_count(a, l, s.t[k], tmax, (double)t_lse, s.z[k], inv);
            l.Z = dt_warp_sum(l.Z), l.A = dt_warp_sum(l.A), l.B = dt_warp_sum(l.B);
            const float loss = dt_loss(a, l, outer.m, (double)outer.s, weight, inv);
            if (lane == 0) a.loss[r] = weight == 0.0f ? 0.0f : loss;
        }
        __syncthreads();
        if (mine) *word = 0;   // (a whole word, by each of its entries)
    }
}

template <typename T, int NV, bool GRAD_ONLY> int dc_launch(s2v_ctx* ctx, cudaStream_t st, const DtArgs& a, int ctas)
{
    const int64_t most = (a.cols / PIECE<T> + ctas - 1) / ctas;
    int64_t rows = a.rows;
    if (rows > (1 << 20)) rows = 1 << 20;   // (clusters; further rows in turns)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * ctas));
    cfg.blockDim = dim3(DC_THREADS);
    cfg.dynamicSmemBytes = (size_t)((most + 3) / 4 * 4);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = GRAD_ONLY ? 0 : 1;
    S2V_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, distill_cluster_kernel<T, NV, GRAD_ONLY>, a, ctas));
    S2V_CHECK_LAUNCH(ctx, "distill_cluster_kernel");
    return S2V_OK;
}
template <typename T, int NV, bool GRAD_ONLY> int dw_launch(s2v_ctx* ctx, cudaStream_t st, const DtArgs& a)
{
    int64_t blocks = (a.rows + DW_WARPS - 1) / DW_WARPS;
    const int64_t cap = (int64_t)ctx->sm_count * 16;
    if (blocks > cap) blocks = cap;
    distill_warp_kernel<T, NV, GRAD_ONLY><<<(unsigned)blocks, 32 * DW_WARPS, 0, st>>>(a);
    S2V_CHECK_LAUNCH(ctx, "distill_warp_kernel");
    return S2V_OK;
}

template <typename T, bool GRAD_ONLY> int dt_launch_type(s2v_ctx* ctx, cudaStream_t st, const DtArgs& a)
{
    const int64_t pieces = a.cols / PIECE<T>;
    if (pieces <= 32) return dw_launch<T, 1, GRAD_ONLY>(ctx, st, a);
    if (pieces <= 32 * DW_PIECES) return dw_launch<T, DW_PIECES, GRAD_ONLY>(ctx, st, a);
    int ctas = 1;
    while (ctas < DC_CTAS && (pieces > (int64_t)ctas * 8 * DC_THREADS || (a.rows * ctas < 2 * ctx->sm_count && pieces >= (int64_t)ctas * 2 * DC_THREADS))) ctas *= 2;
    const int64_t most = (pieces + ctas - 1) / ctas;
    if (most <= 2 * DC_THREADS) return dc_launch<T, 2, GRAD_ONLY>(ctx, st, a, ctas);
    if (most <= 4 * DC_THREADS) return dc_launch<T, 4, GRAD_ONLY>(ctx, st, a, ctas);
    return dc_launch<T, 8, GRAD_ONLY>(ctx, st, a, ctas);
}
int dt_launch(s2v_ctx* ctx, s2v_stream stream, int z_type, bool grad_only, const DtArgs& a)
{
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    return s2v_by_dtype(z_type, [&](auto type) {
        using T = decltype(type);
        return grad_only ? dt_launch_type<T, true>(ctx, st, a) : dt_launch_type<T, false>(ctx, st, a);
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
