// Distillation: Kullback-Leibler loss of a student's logits against a teacher's top logits, and its gradient.
//
// The listed columns and all others are summed apart, each relative to its own largest z: S_in = sum of exp((z - M_in) / T) over the list,
// S_out the same over the rest.  With M the larger maximum and total = S_in exp((M_in - M) / T) + S_out exp((M_out - M) / T),
//     log q_j = (z_j - M) / T - log total,     log s = -log(1 + exp(d)),  d = log(S_in / S_out) + (M_in - M_out) / T.
// Taking one sum from the other's total would lose s (or 1 - s) where the student gives nearly everything (or nothing) to the list, and one
// maximum for both would lose the smaller sum where they are far apart (logits masked with the type's lowest value).  The loss is put together in 64
// bits (it is a difference of larger numbers), and so are the list's p, of whose sum little may be left; the sums over columns and the gradient in fp32.
#include <algorithm>

#include "elem_types.cuh"

namespace
{

constexpr int DT_TOP = 256;            // most entries of a list
constexpr int64_t DT_ROW_BYTES = 1 << 20;   // longest rows: eight runs
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
    double inv;       // 1 / temperature
    float inv_t, c;   // the same; log2 e / temperature
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
// The largest of the teacher's logits: NaN where one of them is, so that a list of NaN is none whose every t is -infinity.
__device__ __forceinline__ float dt_nan_max(float a, float b)
{
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
__device__ __forceinline__ float dt_warp_nan_max(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v = dt_nan_max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// ---------------------------------------------------------------- sums and gradients of pieces of 16 bytes
__device__ __forceinline__ uint64_t dt_two(float a, float b)
{
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void dt_halves(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t dt_add2(uint64_t a, uint64_t b)
{
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t dt_mul2(uint64_t a, uint64_t b)
{
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
// exp2((x + minus_m) * c) of two numbers
__device__ __forceinline__ uint64_t dt_exp_two(float x0, float x1, uint64_t minus_m, uint64_t c)
{
    float a, b;
    dt_halves(dt_mul2(dt_add2(dt_two(x0, x1), minus_m), c), a, b);
    return dt_two(dt_exp2(a), dt_exp2(b));
}

// The largest elements of pieces, lane by lane of the register; then of a register's own.  (NaN loses here and shows in the sums.)
__device__ __forceinline__ uint32_t dt_max_word(uint32_t a, uint32_t b, float) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
__device__ __forceinline__ uint32_t dt_max_word(uint32_t a, uint32_t b, __half)
{
    const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t dt_max_word(uint32_t a, uint32_t b, __nv_bfloat16)
{
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
template <typename T> __device__ __forceinline__ uint32_t dt_max_piece(const uint4& v) { return dt_max_word(dt_max_word(v.x, v.y, T()), dt_max_word(v.z, v.w, T()), T()); }
__device__ __forceinline__ float dt_max_of_word(uint32_t a, float) { return __uint_as_float(a); }
__device__ __forceinline__ float dt_max_of_word(uint32_t a, __half) { return fmaxf(__half2float(__ushort_as_half((unsigned short)a)), __half2float(__ushort_as_half((unsigned short)(a >> 16)))); }
__device__ __forceinline__ float dt_max_of_word(uint32_t a, __nv_bfloat16) { return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u)); }
template <typename T> __device__ __forceinline__ uint32_t dt_lowest()   // a register of -infinity
{
    return sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
}
// -infinity in the place of the listed elements
template <typename T> __device__ __forceinline__ void dt_take_out(uint4& v, uint32_t listed)
{
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            if (listed >> i & 1) w[i] = dt_lowest<T>();
        } else {
            if (listed >> (2 * i) & 1) w[i] = (w[i] & 0xffff0000u) | (dt_lowest<T>() & 0xffffu);
            if (listed >> (2 * i + 1) & 1) w[i] = (w[i] & 0xffffu) | (dt_lowest<T>() & 0xffff0000u);
        }
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
}

struct DtSum {   // of exp((z - m) / T), relative to the largest z
    float m, s;
    __device__ __forceinline__ void reach(float top, float c)
    {
        if (top > m) {
            s *= dt_exp2((m - top) * c);   // (m = -infinity: no sum yet)
            m = top;
        }
    }
    template <typename T> __device__ __forceinline__ void add_piece(const uint4& v, uint64_t minus_m, uint64_t c, uint64_t& sum)   // (m is reached)
    {
        constexpr int N = PIECE<T>;
        float x[N];
        unpack_piece(v, x, T());
#pragma unroll
        for (int i = 0; i < N; i += 2) sum = dt_add2(sum, dt_exp_two(x[i], x[i + 1], minus_m, c));
    }
    // pieces in registers, one of their own at a time for the others (`n` of them in all)
    template <typename T, int NV> __device__ __forceinline__ void add_pieces(const uint4 (&v)[NV], int at, int step, int n, float c)
    {
        uint32_t top = dt_lowest<T>();
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * step + at < n) top = dt_max_word(top, dt_max_piece<T>(v[j]), T());
        reach(dt_max_of_word(top, T()), c);
        const float base = -dt_finite_or_zero(m);
        const uint64_t base2 = dt_two(base, base), c2 = dt_two(c, c);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * step + at < n) add_piece<T>(v[j], base2, c2, sum[j & 1]);
        float a, b;
        dt_halves(dt_add2(sum[0], sum[1]), a, b);
        s += a + b;
    }
    __device__ __forceinline__ void add_one(float x, float c)
    {
        reach(x, c);
        s += dt_exp2((x - dt_finite_or_zero(m)) * c);
    }
    // joined over groups of LANES lanes
    template <int LANES> __device__ __forceinline__ void join(float c)
    {
        float top = m;
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        s *= dt_exp2((m - dt_finite_or_zero(top)) * c);
        m = top;
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
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

// gradient of a piece; what is listed of it is written over by its entry
template <typename T> __device__ __forceinline__ void dt_store(T* to, bool whole, const uint4& v, uint64_t minus_m, uint64_t outer, uint64_t c)
{
    constexpr int N = PIECE<T>;
    float x[N], e[N];
    unpack_piece(v, x, T());
#pragma unroll
    for (int i = 0; i < N; i += 2) dt_halves(dt_mul2(dt_exp_two(x[i], x[i + 1], minus_m, c), outer), e[i], e[i + 1]);
    if (whole) {
        __stcs(reinterpret_cast<uint4*>(to), pack_piece(e, T()));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = from_f32<T>(e[i]);
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
__device__ __forceinline__ void dt_count(const DtArgs& a, DtList& l, double P, float tv, float tmax, double t_lse, float zk, double inv_t)
{
    const double lp = dt_log_p(a, tv, tmax, t_lse, inv_t);
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
// 1 - sum P is taken in 64 bits; what is made of it in fp32 are factors, each off by a few 2^-24 of itself (outer: of its larger term, both are parts of the gradient).
__device__ __forceinline__ DtCoef dt_coefficients(const DtArgs& a, double Z, const DtSum& in, const DtSum& out, float weight, float inv_t, float c)
{
    DtCoef k;
    const float m = fmaxf(in.m, out.m);
    k.M = dt_finite_or_zero(m);
    const float e_out = out.s == 0.0f ? 0.0f : dt_exp2((out.m - k.M) * c), e_in = in.s == 0.0f ? 0.0f : dt_exp2((in.m - k.M) * c);
    const float total = m == -INFINITY ? NAN : in.s * e_in + out.s * e_out;
    float given, rest;
    if (a.t_lse) {
        given = (float)(Z + (Z - Z));     // (infinite: NaN)
        rest = Z > 1.0 ? 0.0f : (float)(1.0 - Z);
        k.p_scale = 1.0f;
    } else {
        given = (float)(Z - Z + 1.0);   // one, and NaN where the list holds NaN or +infinity
        rest = 0.0f;
        k.p_scale = 1.0f / (float)Z;
    }
    k.scale = weight * inv_t;
    const float both = __fdividef(given + rest, total);
    k.inner = k.scale * both;
    k.outer = k.scale * (out.s == 0.0f && both == both ? 0.0f : both * e_out - __fdividef(rest, out.s));
    return k;
}
// (A warp's work, all lanes with the same arguments: its logarithms are taken side by side in three lanes.)
__device__ __forceinline__ float dt_loss(const DtArgs& a, const DtList& l, const DtSum& out, float weight, double inv_t, float c)
{
    const float mf = fmaxf(l.m, out.m), M = dt_finite_or_zero(mf);
    const double in_part = l.s == 0.0 ? 0.0 : l.s * (double)dt_exp2((l.m - M) * c), out_part = out.s == 0.0f ? 0.0 : (double)out.s * (double)dt_exp2((out.m - M) * c);
    const double total = in_part + out_part;   // at least one, where there is a finite z
    const double rest = !a.t_lse || l.Z > 1.0 ? 0.0 : 1.0 - l.Z;
    const double odds = in_part / out_part;    // of the list against the others: log s = -log(1 + odds)
    const int lane = threadIdx.x & 31;
    const double log1 = log1p(lane == 0 ? total - 1.0 : lane == 1 ? odds : a.t_lse ? -l.Z : l.Z - 1.0);
    const double lse = __shfl_sync(0xffffffffu, log1, 0), log_z = __shfl_sync(0xffffffffu, log1, 2);
    double minus_log_s = __shfl_sync(0xffffffffu, log1, 1);
    // sum of p (log p - log q), log q = (z - M) / T - lse; B is relative to l.m
    const double from = l.m == -INFINITY ? 0.0 : ((double)l.m - (double)M) * inv_t, B = l.B + l.Z * from;
    double kl = a.t_lse ? l.A - B + l.Z * lse : (l.A - B) / l.Z - log_z + lse;
    if (rest != 0.0) {
        if (!(odds < 1e30)) minus_log_s = log(l.s / (double)out.s) + ((double)l.m - (double)out.m) * inv_t;   // (too far apart for fp32; 1 / odds is nothing)
        if (out.s != 0.0f) kl += rest * (log_z + minus_log_s);
        else if (rest > 1.0 / 65536.0) kl = INFINITY;
    }
    if (mf == -INFINITY || !(l.Z < INFINITY)) kl = NAN;
    return (float)(kl * weight);
}

// ---------------------------------------------------------------- rows of up to 512 pieces: a warp each
// The row stays in registers between the sums and the gradient.  (16384 x 2500 bf16 by CTAs of 128 threads: 153 us.)
constexpr int DW_WARPS = 4, DW_PIECES = 16;   // pieces a lane, at most
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
    const double inv = a.inv;
    const float inv_t = a.inv_t, c = a.c;
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
            tmax = dt_nan_max(tmax, dt_load_t(a, r, k));
        }
        some = __any_sync(0xffffffffu, some);
        tmax = dt_warp_nan_max(tmax);
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
                if (j * 32 + lane < row.pieces)
                    if (const uint32_t listed = mask[j * 32 + lane]) dt_take_out<T>(v[j], listed);
            outer.template add_pieces<T, NV>(v, lane, 32, row.pieces, c);
            if (!edge_listed) outer.add_one(edge, c);
            outer.template join<32>(c);
            if (a.stats && lane == 0) reinterpret_cast<float4*>(a.stats)[r] = make_float4(outer.m, outer.s, inner.m, inner.s);
            const float loss = dt_loss(a, l, outer, weight, inv, c);
            if (lane == 0) a.loss[r] = weight == 0.0f ? 0.0f : loss;
        }
        if (dz && weight == 0.0f) {   // (for the stats alone)
            __syncwarp();
            dt_zero_row(dz, a.cols, lane, 32);
        } else if (dz) {
            const DtCoef k = dt_coefficients(a, l.Z, inner, outer, weight, inv_t, c);
            const float base = dt_finite_or_zero(outer.m);
            T* const dp = dz + row.head;
            const bool whole = (reinterpret_cast<uintptr_t>(dp) & 15) == 0;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (j * 32 + lane < row.pieces) dt_store(dp + (j * 32 + lane) * N, whole, v[j], dt_two(-base, -base), dt_two(k.outer, k.outer), dt_two(c, c));
            if (!edge_listed) dz[edge_at] = from_f32<T>(dt_exp2((edge - base) * c) * k.outer);
            __syncwarp();   // the listed columns have been written as the others
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

// ---------------------------------------------------------------- longer rows: a CTA or a cluster of CTAs each
// Every CTA has an equal run of the row's pieces.  The first `held` of them lie in shared memory between the sums and the gradient, the others are
// read once more, from L2.  Several CTAs share an SM, so that some move data while others join sums or wait.  Listed columns become -infinity in shared
// memory; the others' are named by a byte per piece.  Their gradients are written over what the loops over the run wrote.  The first CTA's first
// warp adds up the loss while the others write the gradient.
constexpr int DC_CTAS = 8, DC_LISTERS = DT_TOP / 32;
// Rows of up to DC_SHORT pieces: CTAs of 128 threads, all held; six an SM up to 1,950 pieces, beyond as many as its shared memory takes, four at DC_SHORT (the steps of
// a row are a chain of latencies, which more CTAs cover better than more threads: 16384 rows of 9000 bf16 with their gradients 159 us, by six CTAs of 256 that hold
// nothing 232, 8192 of 20000 159 and 162; the two meet at 2,800 pieces, 8192 of 23900 188 and 178).  Lists of more than 128 entries apart.  Longer ones,
// where a CTA takes a row and there are more of them than run at a time: six of 256 threads, nothing held (8192 rows of 32768 bf16 217 us; three that hold 4000 pieces 245).  Rows of more than DC_RUN pieces, and
// few rows: three of 256 that hold 4000 pieces (4096 rows of 131072 bf16 470 us; six that hold none 483, six of 128 562, two of 512 620 to 650, all
// pieces held by a cluster of four 504).
// The loss alone, of rows of more than DC_ONCE pieces and more of them than run at a time, needs a row once: nothing is held, eight CTAs of 128 threads or
// six of 256 an SM (4096 rows of 131072 bf16 202 us, 5.3 TB/s, held 282; of 20000 57 and 76; 8192 of 16384 89 and 96, of 14000 87 and 82).
constexpr int DC_SHORT = 3000, DC_ONCE = 1900, DC_HELD = 4000, DC_RUN = 8192;   // pieces: of short rows; of rows held all the same; held, and of a run, at most
constexpr int DC_SMEM = 72 << 10;
static_assert(DC_HELD * 16 + (DC_RUN - DC_HELD) <= DC_SMEM && DC_SHORT <= DC_HELD, "a byte for each piece that is not held");
constexpr int DC_SLOTS = 512;                        // of the table that finds columns listed twice
struct DcShared {
    double P[DT_TOP], Z[DC_LISTERS];
    union {
        int slot[DC_SLOTS];
        float z[DT_TOP];   // (once the table has been used)
    };
    float t[DT_TOP];
    int id[DT_TOP];
    float4 peer[DC_CTAS];      // outer and inner sums of the cluster's CTAs
    float2 outer[16], inner[DC_LISTERS];
    float tmax[DC_LISTERS];
    int has[DC_LISTERS];       // bit 0: an entry; bit 1: a column that is listed twice
};

// what a row's threads load first: their entry, the row's weight and normaliser
struct DcHead {
    int id;
    float t, weight, t_lse;
    __device__ __forceinline__ DcHead(const DtArgs& a, int64_t r) : id(-1), t(-INFINITY)
    {
        weight = a.row_weight ? __ldg(a.row_weight + r) : 1.0f;
        t_lse = a.t_lse ? __ldg(a.t_lse + r) : 0.0f;
        if (threadIdx.x < a.top) {
            id = dt_load_id(a, r, threadIdx.x);
            t = dt_load_t(a, r, threadIdx.x);
        }
    }
};
// What every thread with an entry knows of it, before z is looked at.
struct DcEntry {
    float t, tmax;
    double P;
    bool twice;   // whether another entry of this column was there first
};
__device__ __forceinline__ DcEntry dc_entry(const DtArgs& a, const DcHead& h, DcShared& s)
{
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool lister = warp * 32 < a.top;   // warps with entries
    DcEntry e{h.id >= 0 ? h.t : -INFINITY, -INFINITY, 0.0, false};
    if (!a.t_lse) {
        if (lister) {
            const float m = dt_warp_nan_max(e.t);
            if (lane == 0) s.tmax[warp] = m;
        }
        __syncthreads();
        for (int w = 0; w * 32 < a.top; ++w) e.tmax = dt_nan_max(e.tmax, s.tmax[w]);
    }
    if (lister) {
        if (h.id >= 0) {
            int was, at = h.id & (DC_SLOTS - 1);   // (twice as many places as entries)
            while ((was = atomicCAS(&s.slot[at], -1, h.id)) != -1 && was != h.id) at = (at + 1) & (DC_SLOTS - 1);
            e.twice = was == h.id;
        }
        s.id[tid] = h.id;
        s.t[tid] = e.t;
        const int has = (__any_sync(0xffffffffu, h.id >= 0) ? 1 : 0) | (__any_sync(0xffffffffu, e.twice) ? 2 : 0);
        if (lane == 0) s.has[warp] = has;
    }
    return e;
}
// The entries' P and their sum, in 64 bits: where the list has nearly everything, the gradient goes by 1 - sum P, and t / T - t_lse in fp32 is off by 2^-24 of |t / T|
// and more (T = 1.5, t around 200, a rest of 1e-4: the gradient of what is not listed by some hundredths of itself).
__device__ __forceinline__ void dc_weigh(const DtArgs& a, const DcHead& h, DcEntry& e, DcShared& s)
{
    if ((threadIdx.x & ~31) >= a.top) return;
    // Nothing of this is done ahead of the row's other loads: converted to 64 bits where it is loaded, the normaliser made every thread wait for it before it asked for
    // the rest (16384 x 9000 bf16 loss 127 us instead of 114, with gradient 169 and 157).
    float t_lse = h.t_lse;
    asm volatile("" : "+f"(t_lse), "+f"(e.t));
    if (h.id >= 0) e.P = exp(dt_log_p(a, e.t, e.tmax, (double)t_lse, a.inv));
    s.P[threadIdx.x] = e.P;
    const double Z = dt_warp_sum(e.P);
    if ((threadIdx.x & 31) == 0) s.Z[threadIdx.x >> 5] = Z;
}
// (after a barrier) bit 0: the row's list has an entry that counts; bit 1: a column is listed twice
__device__ __forceinline__ int dc_has(const DtArgs& a, const DcEntry& e, const DcShared& s)
{
    int has = 0;
    for (int w = 0; w * 32 < a.top; ++w) has |= s.has[w];
    return !a.t_lse && e.tmax == -INFINITY ? has & 2 : has;
}
// Where some column is listed twice: whether an entry is the first of its column; P of all of the column's.
__device__ __forceinline__ bool dc_first(const DtArgs& a, int id, const DcShared& s, float& P)
{
    bool first = true;
    double sum = 0.0;
    for (int k = 0; k < a.top; ++k)
        if (s.id[k] == id) {
            sum += s.P[k];
            if (k < (int)threadIdx.x) first = false;
        }
    P = (float)sum;
    return first;
}
__device__ __forceinline__ double dc_Z(const DtArgs& a, const DcShared& s)
{
    double Z = 0.0;
    for (int w = 0; w * 32 < a.top; ++w) Z += s.Z[w];
    return Z;
}

// where a CTA's run lies
template <typename T> struct DcRun {
    row_pieces<T> row;
    int first, pieces;   // pieces of the run
    __device__ __forceinline__ DcRun(const T* z, int64_t cols, int rank, int ctas) : row(z, cols)
    {
        const int most = (int)((cols / PIECE<T> + ctas - 1) / ctas);
        first = rank * most;
        pieces = max(0, min(most, row.pieces - first));
    }
    // whether a column belongs to this CTA (the head to the first, the tail to the last), and its place among the run's elements, or -1 (head, tail)
    __device__ __forceinline__ bool has(int id, int rank, int ctas, int& at) const
    {
        const int e = id - row.head;
        at = -1;
        if (id < 0) return false;
        if (e < 0) return rank == 0;
        if (e >= row.pieces * PIECE<T>) return rank == ctas - 1;
        at = e - first * PIECE<T>;
        return at >= 0 && at < pieces * PIECE<T>;
    }
};

template <typename T, int DC_THREADS, int CTAS_SM, bool LOSS>
__global__ void __launch_bounds__(DC_THREADS, CTAS_SM) distill_cluster_kernel(const DtArgs a, int ctas, int held)
{
    extern __shared__ __align__(16) unsigned char dc_raw[];
    __shared__ DcShared s;
    constexpr int N = PIECE<T>, DC_WARPS = DC_THREADS / 32;
    uint4* const run = reinterpret_cast<uint4*>(dc_raw);
    const int unmarked = LOSS ? 0 : held;
    uint32_t* const marks = reinterpret_cast<uint32_t*>(run + unmarked);       // a byte for each piece behind those
    const uint8_t* const mark = reinterpret_cast<const uint8_t*>(marks) - unmarked;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)(blockIdx.x % (unsigned)ctas);
    if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // (this CTA has started: the others may write its shared memory)
    const double inv = a.inv;
    const float inv_t = a.inv_t, c = a.c;
    const int most = (int)((a.cols / N + ctas - 1) / ctas);
    for (int w = tid; w < (most - unmarked + 3) / 4; w += DC_THREADS) marks[w] = 0;
    for (int w = tid; w < DC_SLOTS; w += DC_THREADS) s.slot[w] = -1;
    if (tid < DC_LISTERS) s.inner[tid] = make_float2(-INFINITY, 0.0f);   // (of the warps without entries, once and for all)
    const int64_t r = blockIdx.x / (unsigned)ctas;
    const T* const z = static_cast<const T*>(a.z) + r * a.ldz;
    T* const dz = !LOSS && a.dz ? static_cast<T*>(a.dz) + r * a.lddz : nullptr;
    const DcHead head(a, r);
    const float weight = head.weight;
    const DcRun<T> my(z, a.cols, rank, ctas);
    const uint4* const zp = reinterpret_cast<const uint4*>(z + my.row.head) + my.first;
    const bool skip_weight = weight == 0.0f && !a.stats;
    const int kept = min(held, my.pieces);
    if (!LOSS && !skip_weight)
        for (int p = tid; p < kept; p += DC_THREADS) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(run + p)), "l"(zp + p) : "memory");
    __syncthreads();   // the table and the marks are empty
    DcEntry e = dc_entry(a, head, s);
    dc_weigh(a, head, e, s);
    int at;
    const bool here = my.has(head.id, rank, ctas, at), held_entry = !LOSS && here && at >= 0 && at < held * N;
    bool mine = here && !e.twice;
    float P_all = (float)e.P, zk = (here && !held_entry) || (rank == 0 && head.id >= 0) ? to_f32(z[head.id]) : -INFINITY;
    if (here && at >= unmarked * N) atomicOr(&marks[(at / N - unmarked) >> 2], 1u << (8 * ((at / N - unmarked) & 3) + at % N));
    // the scalar columns: the head's to the first CTA, the tail's to the last
    const bool in_head = rank == 0 && tid < my.row.head, in_tail = rank == ctas - 1 && tid >= 32 && tid < 32 + my.row.tail;
    const int edge_at = in_head ? tid : (int)a.cols - my.row.tail + tid - 32;
    const float edge = in_head || in_tail ? to_f32(z[edge_at]) : -INFINITY;
    __syncthreads();
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int has = dc_has(a, e, s);
    if (skip_weight || !(has & 1)) {   // (the same for all CTAs of the row)
        if (rank == 0) {
            if (tid == 0) a.loss[r] = 0.0f;
            if (a.stats && tid < 4) a.stats[4 * r + tid] = 0.0f;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();   // (dz may be z)
        if (dz) dt_zero_row(dz, a.cols, rank * DC_THREADS + tid, ctas * DC_THREADS);
        return;
    }
    bool edge_out = in_head || in_tail;   // not listed
    if (edge_out)
        for (int k = 0; k < a.top; ++k) edge_out &= s.id[k] != edge_at;
    if ((has & 2) && here) mine = dc_first(a, head.id, s, P_all);
    DtSum outer{-INFINITY, 0.0f}, inner{-INFINITY, 0.0f};
    const auto add = [&](int from, int n) {
        for (int p = from + tid; p < n; p += 4 * DC_THREADS) {
            uint4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (p + j * DC_THREADS < n) v[j] = zp[p + j * DC_THREADS];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (p + j * DC_THREADS < n)
                    if (const uint32_t listed = mark[p + j * DC_THREADS]) dt_take_out<T>(v[j], listed);
            outer.template add_pieces<T, 4>(v, p, DC_THREADS, n, c);
        }
    };
    add(held, my.pieces);   // what is not held, while the rest is on its way
    if constexpr (LOSS) add(0, kept);   // (in the same order, and the same loss to the last bit, as with a gradient)
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    if (mine && held_entry) {   // (one thread an element)
        T* const element = reinterpret_cast<T*>(run) + at;
        zk = to_f32(*element);
        *element = from_f32<T>(-INFINITY);
    }
    if (warp * 32 < a.top) {
        s.z[tid] = zk;
        // (a listed z of -infinity adds nothing, +infinity and NaN make the sum NaN)
        if (mine) inner = DtSum{zk, zk < INFINITY ? zk > -INFINITY ? 1.0f : 0.0f : NAN};
        inner.template join<32>(c);
        if (lane == 0) s.inner[warp] = make_float2(inner.m, inner.s);
    }
    __syncthreads();
    for (int p = tid; !LOSS && p < kept; p += 4 * DC_THREADS) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (p + j * DC_THREADS < kept) v[j] = run[p + j * DC_THREADS];
        outer.template add_pieces<T, 4>(v, p, DC_THREADS, kept, c);
    }
    if (edge_out) outer.add_one(edge, c);
    outer.template join<32>(c);
    if (lane == 0) s.outer[warp] = make_float2(outer.m, outer.s);
    __syncthreads();
    if (warp == 0) {   // the CTA's sums: lanes 0 to 15 the outer ones, 16 to 23 the inner ones
        const float2 o = lane < DC_WARPS ? s.outer[lane] : lane >= 16 && lane < 16 + DC_LISTERS ? s.inner[lane - 16] : make_float2(-INFINITY, 0.0f);
        DtSum d{o.x, o.y};
        d.template join<16>(c);
        const float m_in = __shfl_sync(0xffffffffu, d.m, 16), s_in = __shfl_sync(0xffffffffu, d.s, 16);
        if (lane < ctas) {
            uint32_t to;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(&s.peer[rank])), "r"(lane));
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(d.m), "f"(d.s), "f"(m_in), "f"(s_in) : "memory");
        }
        __syncwarp();
    }
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
    {
        const float4 o = (lane & 7) < ctas ? s.peer[lane & 7] : make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
        DtSum d = lane & 8 ? DtSum{o.z, o.w} : DtSum{o.x, o.y};
        d.template join<8>(c);
        outer = DtSum{__shfl_sync(0xffffffffu, d.m, 0), __shfl_sync(0xffffffffu, d.s, 0)};
        inner = DtSum{__shfl_sync(0xffffffffu, d.m, 8), __shfl_sync(0xffffffffu, d.s, 8)};
    }
    if (a.stats && rank == 0 && tid == DC_THREADS - 1) reinterpret_cast<float4*>(a.stats)[r] = make_float4(outer.m, outer.s, inner.m, inner.s);
    if (dz && weight == 0.0f) {   // (for the stats alone; the cluster has read the row)
        dt_zero_row(dz, a.cols, rank * DC_THREADS + tid, ctas * DC_THREADS);
    } else if (dz) {
        const DtCoef k = dt_coefficients(a, dc_Z(a, s), inner, outer, weight, inv_t, c);
        const float base = dt_finite_or_zero(outer.m);
        const uint64_t base2 = dt_two(-base, -base), outer2 = dt_two(k.outer, k.outer), c2 = dt_two(c, c);
        T* const dp = dz + my.row.head + (int64_t)my.first * N;
        const bool whole = (reinterpret_cast<uintptr_t>(dp) & 15) == 0;
        for (int p = held + tid; p < my.pieces; p += 4 * DC_THREADS) {
            uint4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (p + j * DC_THREADS < my.pieces) v[j] = zp[p + j * DC_THREADS];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (p + j * DC_THREADS < my.pieces) dt_store(dp + (p + j * DC_THREADS) * N, whole, v[j], base2, outer2, c2);
        }
        if (whole) {
#pragma unroll 4
            for (int p = tid; p < kept; p += DC_THREADS) dt_store(dp + p * N, true, run[p], base2, outer2, c2);
        } else {
            for (int p = tid; p < kept; p += DC_THREADS) dt_store(dp + p * N, false, run[p], base2, outer2, c2);
        }
        if (edge_out) dz[edge_at] = from_f32<T>(dt_exp2((edge - base) * c) * k.outer);
        __syncthreads();   // the listed columns have been written as the others
        if (mine) dz[head.id] = from_f32<T>(k.inner * expf((zk - k.M) * inv_t) - k.scale * (P_all * k.p_scale));
    }
    if (rank == 0 && warp == 0) {
        DtList l{0.0, 0.0, 0.0, (double)inner.s, inner.m};
        for (int k = lane; k < a.top; k += 32)
            if (s.id[k] >= 0) dt_count(a, l, s.P[k], s.t[k], e.tmax, (double)head.t_lse, s.z[k], inv);
        l.Z = dt_warp_sum(l.Z), l.A = dt_warp_sum(l.A), l.B = dt_warp_sum(l.B);
        const float loss = dt_loss(a, l, outer, weight, inv, c);
        if (lane == 0) a.loss[r] = weight == 0.0f ? 0.0f : loss;
    }
}

// The gradient from kept sums: nothing to wait for but the list.
// (CTAs of 128 threads up to 4096 pieces a row, else of 256: 16384 x 9000 bf16 116 us, with 256 threads 177 and with 512 282.  Long rows in several runs:
// 4096 x 131072 bf16 337 us, 6.4 TB/s, a CTA a row 347, four CTAs 454; 483 x 186542 fp32 121 and 140; 1300 x 131072 fp32 215 and 232.)
template <typename T, int DG_THREADS> __global__ void __launch_bounds__(DG_THREADS, 1024 / DG_THREADS) distill_grad_kernel(const DtArgs a, int ctas)
{
    __shared__ DcShared s;
    constexpr int N = PIECE<T>;
    const int tid = threadIdx.x;
    const int rank = (int)(blockIdx.x % (unsigned)ctas);
    const float inv_t = a.inv_t, c = a.c;
    for (int w = tid; w < DC_SLOTS; w += DG_THREADS) s.slot[w] = -1;
    const int64_t r = blockIdx.x / (unsigned)ctas;
    const T* const z = static_cast<const T*>(a.z) + r * a.ldz;
    T* const dz = static_cast<T*>(a.dz) + r * a.lddz;
    const DcHead head(a, r);
    const float weight = head.weight;
    const float4 st = __ldg(reinterpret_cast<const float4*>(a.stats) + r);
    const DcRun<T> my(z, a.cols, rank, ctas);
    int at;
    const bool here = my.has(head.id, rank, ctas, at);
    const float zk = here ? to_f32(z[head.id]) : 0.0f;   // (on its way under the exponentials)
    const bool in_head = rank == 0 && tid < my.row.head, in_tail = rank == ctas - 1 && tid >= 32 && tid < 32 + my.row.tail;
    const int edge_at = in_head ? tid : (int)a.cols - my.row.tail + tid - 32;
    const float edge = in_head || in_tail ? to_f32(z[edge_at]) : 0.0f;
    __syncthreads();   // the table is empty
    DcEntry e = dc_entry(a, head, s);
    dc_weigh(a, head, e, s);
    bool mine = here && !e.twice;
    float P_all = (float)e.P;
    // (the barrier also stands between the reads of listed columns and the writes: dz may be z)
    __syncthreads();
    const int has = dc_has(a, e, s);
    if ((has & 2) && here) mine = dc_first(a, head.id, s, P_all);
    if (weight == 0.0f || !(has & 1)) {
        dt_zero_row(dz, a.cols, rank * DG_THREADS + tid, ctas * DG_THREADS);
        return;
    }
    const DtSum outer{st.x, st.y}, inner{st.z, st.w};
    const DtCoef k = dt_coefficients(a, dc_Z(a, s), inner, outer, weight, inv_t, c);
    const float base = dt_finite_or_zero(outer.m);
    const uint64_t base2 = dt_two(-base, -base), outer2 = dt_two(k.outer, k.outer), c2 = dt_two(c, c);
    const uint4* const zp = reinterpret_cast<const uint4*>(z + my.row.head) + my.first;
    T* const dp = dz + my.row.head + (int64_t)my.first * N;
    const bool whole = (reinterpret_cast<uintptr_t>(dp) & 15) == 0;
    for (int p = tid; p < my.pieces; p += 4 * DG_THREADS) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (p + j * DG_THREADS < my.pieces) v[j] = zp[p + j * DG_THREADS];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (p + j * DG_THREADS < my.pieces) dt_store(dp + (p + j * DG_THREADS) * N, whole, v[j], base2, outer2, c2);
    }
    if (in_head || in_tail) dz[edge_at] = from_f32<T>(dt_exp2((edge - base) * c) * k.outer);
    __syncthreads();   // the listed columns have been written as the others
    if (mine) dz[head.id] = from_f32<T>(k.inner * expf((zk - k.M) * inv_t) - k.scale * (P_all * k.p_scale));
}

template <typename T, int THREADS, int CTAS_SM, bool LOSS> int dc_launch(s2v_ctx* ctx, cudaStream_t st, const DtArgs& a, int ctas, int held)
{
    const int64_t most = (a.cols / PIECE<T> + ctas - 1) / ctas;
    const auto kernel = distill_cluster_kernel<T, THREADS, CTAS_SM, LOSS>;
    S2V_CUDA_OK(ctx, s2v_allow_shared(kernel, DC_SMEM));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * ctas));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = LOSS ? (size_t)(most + 3) / 4 * 4 : (size_t)(held * 16 + (most - held + 3) / 4 * 4);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    S2V_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, kernel, a, ctas, held));
    S2V_CHECK_LAUNCH(ctx, "distill_cluster_kernel");
    return S2V_OK;
}
template <typename T, int THREADS> int dg_launch(s2v_ctx* ctx, cudaStream_t st, const DtArgs& a, int ctas)
{
    distill_grad_kernel<T, THREADS><<<(unsigned)(a.rows * ctas), THREADS, 0, st>>>(a, ctas);
    S2V_CHECK_LAUNCH(ctx, "distill_grad_kernel");
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
    if (pieces <= 32 * 8) return dw_launch<T, 8, GRAD_ONLY>(ctx, st, a);
    if (pieces <= 32 * DW_PIECES) return dw_launch<T, DW_PIECES, GRAD_ONLY>(ctx, st, a);
    if (a.rows > INT32_MAX / DC_CTAS) return s2v_fail(ctx, S2V_ERR_UNSUPPORTED, "distill_topk: more than 2^28 rows of this length");
    int ctas = 1;
    if constexpr (GRAD_ONLY) {
        // CTAs for all SMs; and eight times as many as run at a time of long rows, so that none is left with the last ones
        const auto runs = [&](int64_t waves, int64_t each) { return a.rows * ctas < waves * ctx->sm_count && pieces >= ctas * each; };
        while (ctas < DC_CTAS && (runs(2, 1024) || runs(32, 8192))) ctas *= 2;
        return pieces <= 2 * DC_SHORT && a.top <= 128 ? dg_launch<T, 128>(ctx, st, a, ctas) : dg_launch<T, 256>(ctx, st, a, ctas);
    } else {
        while (ctas < DC_CTAS && (pieces > (int64_t)ctas * DC_RUN || (a.rows * ctas < 2 * ctx->sm_count && pieces >= (int64_t)ctas * 512))) ctas *= 2;
        const bool many = a.rows * ctas >= 3 * ctx->sm_count, once = !a.dz && pieces > DC_ONCE && many;
        const int held = (int)std::min<int64_t>(DC_HELD, (pieces + ctas - 1) / ctas);
        if (pieces <= DC_SHORT && a.top <= 128) return once ? dc_launch<T, 128, 8, true>(ctx, st, a, ctas, held) : dc_launch<T, 128, 6, false>(ctx, st, a, ctas, held);
        if (many && ctas == 1) return once ? dc_launch<T, 256, 6, true>(ctx, st, a, 1, 0) : dc_launch<T, 256, 6, false>(ctx, st, a, 1, 0);
        return once ? dc_launch<T, 256, 6, true>(ctx, st, a, ctas, held) : dc_launch<T, 256, 3, false>(ctx, st, a, ctas, held);
    }
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
    const auto bad = [&](int status, const char* what) { return s2v_fail(ctx, status, std::string(name) + ": " + what); };
    if (a.rows < 0 || a.cols <= 0 || a.top <= 0) return bad(S2V_ERR_INVALID_ARG, "negative or empty size");
    if (!s2v_dtype_ok(z_type) || !s2v_dtype_ok(a.t_type)) return bad(S2V_ERR_INVALID_ARG, "unknown element type");
    if (!(a.temperature >= 1e-30f && a.temperature <= 1e30f)) return bad(S2V_ERR_INVALID_ARG, "temperature outside [1e-30, 1e30]");
    if (a.rows == 0) return S2V_OK;
    if (!a.z || !a.idx || !a.t) return bad(S2V_ERR_INVALID_ARG, "NULL pointer");
    if (a.top > DT_TOP) return bad(S2V_ERR_UNSUPPORTED, "more than 256 entries a row");
    if (a.cols > DT_ROW_BYTES / (int64_t)s2v_dtype_bytes(z_type)) return bad(S2V_ERR_UNSUPPORTED, "rows of more than 1,048,576 bytes");
    if (a.rows > 1 && (a.ldz < a.cols || a.ldt < a.top || (a.dz && a.lddz < a.cols)))
        return bad(S2V_ERR_INVALID_ARG, "leading dimension below the number of columns");
    const size_t es = s2v_dtype_bytes(z_type);
    if (reinterpret_cast<uintptr_t>(a.z) % es || reinterpret_cast<uintptr_t>(a.dz) % es || reinterpret_cast<uintptr_t>(a.t) % s2v_dtype_bytes(a.t_type) ||
        !s2v_aligned4(a.idx, a.t_lse, a.row_weight, a.loss))
        return bad(S2V_ERR_INVALID_ARG, "misaligned pointer");
    if (!s2v_aligned16(a.stats)) return bad(S2V_ERR_INVALID_ARG, "stats must be 16-byte aligned");
    if (a.dz == a.z && a.rows > 1 && a.lddz != a.ldz) return bad(S2V_ERR_INVALID_ARG, "dz in the place of z needs the same leading dimension");
    return S2V_OK;
}

}  // namespace

extern "C" {

int s2v_distill_topk(s2v_ctx* ctx, s2v_stream stream, int64_t rows, int64_t cols, int z_type, const void* z, int64_t ldz, int top, const int32_t* idx,
                     int t_type, const void* t, int64_t ldt, const float* t_lse, float temperature, const float* row_weight, float* loss, float* stats,
                     void* dz, int64_t lddz)
{
    S2V_ENTER(ctx);
    const DtArgs a{rows, cols, ldz, ldt, lddz, z, idx, t, t_lse, row_weight, loss, stats, dz, ctx->dstatus_dev, temperature, top, t_type, 1.0 / (double)temperature, 1.0f / temperature, 1.4426950408889634f / temperature};
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
    const DtArgs a{rows, cols, ldz, ldt, lddz, z, idx, t, t_lse, row_weight, nullptr, const_cast<float*>(stats), dz, ctx->dstatus_dev, temperature, top, t_type, 1.0 / (double)temperature, 1.0f / temperature, 1.4426950408889634f / temperature};
    const int rc = dt_check(ctx, "distill_topk_grad", z_type, a);
    if (rc != S2V_OK || rows == 0) return rc;
    if (!stats || !dz) return s2v_fail(ctx, S2V_ERR_INVALID_ARG, "distill_topk_grad: NULL pointer");
    return dt_launch(ctx, stream, z_type, true, a);
}

}  // extern "C"
