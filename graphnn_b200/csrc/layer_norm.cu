// Layer norm of rows, its gradient, and the 8-bit rows that a training step keeps between the two instead of its input.
//
// Forward: a row by 8 lanes, a warp or a CTA, held in registers between its moments and its outputs.  Deviations are summed around the mean of the lanes or the warp,
// and a CTA's warps joined by  sum (x - mean)^2 = sum over warps of (M2_w + n_w (mean_w - mean)^2),  so that one barrier a row gives both moments, without the
// cancellation of E x^2 - (E x)^2.
// Gradient: the same places of a row in every turn of a thread, which so sums its columns of the weight's and the bias's gradient in registers over all
// the rows that it takes; a CTA leaves one line of sums, and a second kernel adds the lines in their order.
#include "f32x2.cuh"
#include "quantize.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace
{

constexpr int LN_CTA = 256;
constexpr int LN_MAX_LINES = 1024;   // CTAs of the gradient, each with a line of column sums in the workspace

// Pieces of a row: 16 bytes where every row lies on a 16-byte boundary, else single elements.
template <typename T, bool VEC> struct ln_piece {
    static constexpr int N = VEC ? 16 / (int)sizeof(T) : 1;
    using raw = typename std::conditional<VEC, uint4, T>::type;
    static __device__ __forceinline__ raw load(const T* row, int64_t p) { return __ldcs(reinterpret_cast<const raw*>(row) + p); }
    static __device__ __forceinline__ raw load_again(const T* row, int64_t p) { return reinterpret_cast<const raw*>(row)[p]; }
    static __device__ __forceinline__ void unpack(const raw& v, float* x)
    {
        if constexpr (VEC) unpack_piece(v, x, T());
        else x[0] = to_f32(v);
    }
    static __device__ __forceinline__ void store(T* row, int64_t p, const float* y)
    {
        if constexpr (VEC) reinterpret_cast<uint4*>(row)[p] = pack_piece(y, T());
        else row[p] = from_f32<T>(y[0]);
    }
    static __device__ __forceinline__ void columns(const float* v, int64_t p, float otherwise, float* w)   // of a vector of fp32, NULL: one value everywhere
    {
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = otherwise;
        if (!v) return;
        if constexpr (VEC) {
            if ((reinterpret_cast<uintptr_t>(v) & 15) == 0) {
#pragma unroll
                for (int e = 0; e < N; e += 4) {
                    const float4 f = __ldg(reinterpret_cast<const float4*>(v + p * N + e));
                    w[e] = f.x, w[e + 1] = f.y, w[e + 2] = f.z, w[e + 3] = f.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) w[e] = __ldg(v + p * N + e);
            }
        } else w[0] = __ldg(v + p);
    }
    static __device__ __forceinline__ uint32_t largest(const raw& v)
    {
        if constexpr (VEC) return q_largest<T>(v);
        else return __float_as_uint(to_f32(v)) & 0x7fffffffu;
    }
    static __device__ __forceinline__ void quantize(int8_t* row, int64_t p, bool whole, const raw& v, const q_row& k)
    {
        if constexpr (VEC) q_store<T>(row + p * N, whole, v, k);
        else row[p] = (int8_t)k.integer(to_f32(v));
    }
    // 8-bit numbers of a piece
    using raw8 = typename std::conditional<VEC, typename std::conditional<N == 8, uint2, uint32_t>::type, int8_t>::type;
    static __device__ __forceinline__ raw8 load8(const int8_t* row, int64_t p) { return __ldcs(reinterpret_cast<const raw8*>(row) + p); }
    static __device__ __forceinline__ void unpack8(const raw8& v, float* x)
    {
        if constexpr (!VEC) x[0] = (float)v;
        else {
            uint32_t w[N / 4];
            if constexpr (N == 8) w[0] = v.x, w[1] = v.y;
            else w[0] = v;
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = (float)(int8_t)(w[e / 4] >> (8 * (e & 3)));
        }
    }
};

template <int LANES> __device__ __forceinline__ float ln_lanes_sum(float v)
{
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Mean and sum of squared deviations of a row from its warps' (sum, sum of squared deviations from the warp's mean) and (1 / count, count): a warp's part a lane.
template <int WARPS> __device__ __forceinline__ void ln_join(const float2* part, const float2* counts, float inv, float& mean, float& m2)
{
    const float2 p = part[threadIdx.x & (WARPS - 1)], c = counts[threadIdx.x & (WARPS - 1)];
    mean = ln_lanes_sum<WARPS>(p.x) * inv;
    const float d = fmaf(p.x, c.x, -mean);
    m2 = ln_lanes_sum<WARPS>(fmaf(d * c.y, d, p.y));
}

// THREADS threads a row (8, 32 or a CTA of THREADS), NV pieces of each in registers; a longer row's others (CTAs alone) are read again.
template <typename T, bool VEC, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS < LN_CTA ? LN_CTA : THREADS)
    layer_norm_kernel(int64_t rows, int64_t cols, const T* x, int64_t ldx, const float* __restrict__ weight, const float* __restrict__ bias, float eps, T* y, int64_t ldy,
                      float2* __restrict__ stats, int8_t* __restrict__ q, int64_t ldq, float* __restrict__ q_scale)   // (y may be x)
{
    using P = ln_piece<T, VEC>;
    constexpr int N = P::N, CTA = THREADS < LN_CTA ? LN_CTA : THREADS, WARPS = THREADS / 32, GROUPS = CTA / THREADS;
    constexpr int LANES = THREADS < 32 ? THREADS : 32;
    __shared__ float2 part[WARPS > 1 ? 2 * WARPS : 1], counts[WARPS > 1 ? WARPS : 1];   // of two turns, so that there is one barrier a row
    __shared__ uint32_t tops[WARPS > 1 ? 2 * WARPS : 1];
    const int at = threadIdx.x % THREADS;
    const int64_t pieces = cols / N;
    const float inv = 1.0f / (float)cols;
    float inv_warp = inv;   // 1 / numbers of the lanes that sum around one mean
    if constexpr (WARPS > 1) {
        const float n = ln_lanes_sum<32>((float)((pieces - at + THREADS - 1) / THREADS * N));
        inv_warp = n > 0.0f ? 1.0f / n : 0.0f;
        if ((at & 31) == 0) counts[at >> 5] = make_float2(inv_warp, n);   // (the first row's barrier is before their first use)
    }
    int turn = 0;
    for (int64_t first = (int64_t)blockIdx.x * GROUPS; first < rows; first += (int64_t)gridDim.x * GROUPS, turn ^= 1) {
        // (groups behind the last row take it too, but leave nothing: all lanes of a warp exchange)
        const int64_t own = first + threadIdx.x / THREADS, r = min(own, rows - 1);
        const bool mine = own < rows;
        const T* const xr = x + r * ldx;
        typename P::raw v[NV];
        float sum = 0.0f, m2 = 0.0f;
        uint32_t a = 0;
        const auto add = [&](const typename P::raw& w) {
            float f[N];
            P::unpack(w, f);
#pragma unroll
            for (int e = 0; e < N; ++e) sum += f[e];
        };
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < pieces) v[j] = P::load_again(xr, j * THREADS + at);
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < pieces) add(v[j]);
        if constexpr (WARPS > 1)
            for (int64_t p = NV * THREADS + at; p < pieces; p += THREADS) add(P::load_again(xr, p));
        sum = ln_lanes_sum<LANES>(sum);
        float mean = sum * inv_warp;
        const auto deviate = [&](const typename P::raw& w) {
            float f[N];
            P::unpack(w, f);
#pragma unroll
            for (int e = 0; e < N; ++e) m2 = fmaf(f[e] - mean, f[e] - mean, m2);
            if (q) a = max(a, P::largest(w));
        };
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < pieces) deviate(v[j]);
        if constexpr (WARPS > 1)
            for (int64_t p = NV * THREADS + at; p < pieces; p += THREADS) deviate(P::load_again(xr, p));
        m2 = ln_lanes_sum<LANES>(m2);
        if (q) {
            if constexpr (THREADS < 32) {
#pragma unroll
                for (int o = THREADS / 2; o; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
            } else a = __reduce_max_sync(0xffffffffu, a);
        }
        if constexpr (WARPS > 1) {
            if ((at & 31) == 0) part[turn * WARPS + (at >> 5)] = make_float2(sum, m2), tops[turn * WARPS + (at >> 5)] = a;
            __syncthreads();
            ln_join<WARPS>(part + turn * WARPS, counts, inv, mean, m2);
            if (q) a = __reduce_max_sync(0xffffffffu, tops[turn * WARPS + (threadIdx.x & (WARPS - 1))]);
        }
        const float rstd = rsqrtf(fmaf(m2, inv, eps));
        if (mine && at == 0 && stats) stats[r] = make_float2(mean, rstd);
        if (!mine) continue;
        T* const yr = y + r * ldy;
        const q_row k(a);
        int8_t* const qr = q + r * ldq;
        const bool whole = VEC && (reinterpret_cast<uintptr_t>(qr) & (N - 1)) == 0;
        const auto leave = [&](int64_t p, const typename P::raw& w) {
            float f[N], g[N], b[N];
            P::unpack(w, f);
            P::columns(weight, p, 1.0f, g);
            P::columns(bias, p, 0.0f, b);
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = fmaf((f[e] - mean) * rstd, g[e], b[e]);
            if (q) P::quantize(qr, p, whole, w, k);
            P::store(yr, p, f);
        };
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < pieces) leave(j * THREADS + at, v[j]);
        if constexpr (WARPS > 1)
            for (int64_t p = NV * THREADS + at; p < pieces; p += THREADS) leave(p, P::load_again(xr, p));
        if (q && at == 0) q_scale[r] = k.scale;
    }
}

// a piece's 8-bit integers from its numbers (of which `largest` is the row's: the same as q_store)
template <int N> __device__ __forceinline__ void q_store_pairs(int8_t* q, bool whole, const uint64_t* x, const q_row& k)
{
    // (the products by single instructions: a packed one and a packed addition behind it are made a multiply-add, whose one rounding gives other integers)
    const uint64_t up = f2_of(12582912.0f, 12582912.0f);
    const auto two = [&](uint64_t v) {
        const float2 f = f2_get(v);
        return f2_get(f2_add(f2_of(__fmul_rn(f.x, k.factor), __fmul_rn(f.y, k.factor)), up));
    };
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const float2 a = two(x[2 * i]), b = two(x[2 * i + 1]);
        w[i] = __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
        if (k.factor == 0.0f) w[i] = 0;
    }
    if (whole) {
        if constexpr (N == 4) *reinterpret_cast<uint32_t*>(q) = w[0];
        else *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) q[e] = (int8_t)(w[e / 4] >> (8 * (e & 3)));
    }
}

// ---- rows through a ring in shared memory
constexpr int LN_STAGES = 8;   // at most

struct ln_ring {
    uint32_t base, full;       // shared addresses: stages, barriers
    unsigned char* at;
    volatile int* abort_flag;
    int stages, bytes;         // of a stage
    __device__ __forceinline__ ln_ring(unsigned char* raw, int stages_, int bytes_) : stages(stages_), bytes(bytes_)
    {
        at = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 127) & ~(uintptr_t)127);
        base = smem_u32(at), full = base + (uint32_t)(stages * bytes);
        abort_flag = reinterpret_cast<volatile int*>(at + stages * bytes + 8 * LN_STAGES);
        if (threadIdx.x == 0) {
            for (int i = 0; i < stages; ++i) tc_mbar_init(full + 8 * i, 1);
            *abort_flag = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
    }
    // by one thread: `n` bytes (a multiple of 16) to a stage, behind `offset`
    __device__ __forceinline__ void copy(int stage, int offset, const void* from, int n) const
    {
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(base + (uint32_t)(stage * bytes + offset)), "l"(from), "r"(n),
                     "r"(full + 8 * stage)
                     : "memory");
    }
    __device__ __forceinline__ bool wait(int stage, uint32_t phase, s2v_device_status* status) const
    {
        const uint32_t bar = full + 8 * stage;
        return __all_sync(0xffffffffu, tc_mbar_try(bar, phase)) || tc_wait(bar, phase, abort_flag, status, 90);
    }
    // where a wait gave up: copies under way, before the CTA goes
    __device__ __forceinline__ void drain(int from, int to) const
    {
        if (threadIdx.x == 0)
            for (int i = from; i < to; ++i) {
                int spins = 0;
                while (!tc_mbar_try(full + 8 * (i % stages), (uint32_t)(i / stages) & 1u))
                    if (++spins > TC_WAIT_LIMIT) break;
            }
    }
    static size_t shared(int stages, int bytes) { return 128 + (size_t)stages * bytes + 8 * LN_STAGES + 16; }
};

struct LnNorm {
    int64_t rows, cols, ldx, ldy, ldq;
    const void* x;
    const float* weight;
    const float* bias;
    float eps;
    void* y;
    float2* stats;
    int8_t* q;
    float* q_scale;
    int stages, bytes;
    s2v_device_status* status;
};

// A row a CTA, NV pieces a thread; one barrier a row, behind which its stage is free.  What a row costs a thread besides its numbers is some 200 instructions, so
// threads are few and pieces many; weight and bias are in registers for all rows.  (8192 x 8192 bf16 with 8-bit rows, threads x pieces x CTAs an SM: 512 x 2 x 1
// 107 us, 256 x 4 x 2 70; 128 x 8 x 5 with weight and bias from L1 92.)
template <typename T, int NV, int THREADS, int CTAS> __global__ void __launch_bounds__(THREADS, CTAS) layer_norm_ring_kernel(const LnNorm a)
{
    using P = ln_piece<T, true>;
    constexpr int N = P::N, WARPS = THREADS / 32;
    __shared__ float2 part[2][WARPS], counts[WARPS];
    __shared__ uint32_t tops[2][WARPS];
    extern __shared__ unsigned char ln_raw[];
    const ln_ring ring(ln_raw, a.stages, a.bytes);
    const int at = threadIdx.x, pieces = (int)(a.cols / N), row_bytes = (int)(a.cols * (int64_t)sizeof(T));
    const int mine = (int)((a.rows - blockIdx.x + gridDim.x - 1) / gridDim.x);   // rows of this CTA
    const auto fetch = [&](int i, int stage) {
        if (i < mine) {
            mbar_expect(ring.full + 8 * stage, (uint32_t)row_bytes);
            ring.copy(stage, 0, static_cast<const T*>(a.x) + ((int64_t)blockIdx.x + (int64_t)i * gridDim.x) * a.ldx, row_bytes);
        }
    };
    if (at == 0)
        for (int i = 0; i < a.stages; ++i) fetch(i, i);
    const float inv = 1.0f / (float)a.cols, n_warp = ln_lanes_sum<32>((float)(max(0, pieces - at + THREADS - 1) / THREADS * N)), inv_warp = n_warp > 0.0f ? 1.0f / n_warp : 0.0f;
    if ((at & 31) == 0) counts[at >> 5] = make_float2(inv_warp, n_warp);   // (the first row's barrier is before their first use)
    uint64_t w[NV * N / 2], b[NV * N / 2];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        float u[N], v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) u[e] = v[e] = 0.0f;
        if (j * THREADS + at < pieces) P::columns(a.weight, j * THREADS + at, 1.0f, u), P::columns(a.bias, j * THREADS + at, 0.0f, v);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) w[j * N / 2 + e] = f2_of(u[2 * e], u[2 * e + 1]), b[j * N / 2 + e] = f2_of(v[2 * e], v[2 * e + 1]);
    }
    int i = 0, stage = 0;
    uint32_t phase = 0;
    bool failed = false;
    for (; i < mine; ++i) {
        const int64_t r = (int64_t)blockIdx.x + (int64_t)i * gridDim.x;
        const bool ok = ring.wait(stage, phase, a.status);
        const uint4* const row = reinterpret_cast<const uint4*>(ring.at + stage * a.bytes);
        uint4 v[NV];
        uint64_t s = 0;   // (two zeros)
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < pieces) {
                v[j] = row[j * THREADS + at];
                uint64_t f[N / 2];
                f2_unpack<T>(v[j], f);
                if (a.q) top = max(top, P::largest(v[j]));
#pragma unroll
                for (int e = 0; e < N / 2; ++e) s = f2_add(s, f[e]);
            }
        const float sum = ln_lanes_sum<32>(f2_sum(s)), near = -sum * inv_warp;
        const uint64_t near2 = f2_of(near, near);
        s = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < pieces) {
                uint64_t f[N / 2];
                f2_unpack<T>(v[j], f);
#pragma unroll
                for (int e = 0; e < N / 2; ++e) {
                    const uint64_t d = f2_add(f[e], near2);
                    s = f2_fma(d, d, s);
                }
            }
        float m2 = ln_lanes_sum<32>(f2_sum(s)), mean;
        if (a.q) top = __reduce_max_sync(0xffffffffu, top);
        if ((at & 31) == 0) part[i & 1][at >> 5] = make_float2(sum, m2), tops[i & 1][at >> 5] = top;
        if (__syncthreads_or(!ok)) {
            failed = true;
            break;
        }
        if (at == 0) fetch(i + a.stages, stage);   // (the row is in registers)
        if (++stage == a.stages) stage = 0, phase ^= 1;
        ln_join<WARPS>(part[i & 1], counts, inv, mean, m2);
        const float rstd = rsqrtf(fmaf(m2, inv, a.eps));
        const uint64_t mean2 = f2_of(-mean, -mean), rstd2 = f2_of(rstd, rstd);
        T* const yr = static_cast<T*>(a.y) + r * a.ldy;
        int8_t* const qr = a.q + r * a.ldq;
        const bool whole = (reinterpret_cast<uintptr_t>(qr) & (N - 1)) == 0;
        const q_row scale(a.q ? __reduce_max_sync(0xffffffffu, tops[i & 1][at & (WARPS - 1)]) : 0u);
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < pieces) {
                uint64_t f[N / 2];
                f2_unpack<T>(v[j], f);
                if (a.q) q_store_pairs<N>(qr + (j * THREADS + at) * N, whole, f, scale);
#pragma unroll
                for (int e = 0; e < N / 2; ++e) f[e] = f2_fma(f2_mul(f2_add(f[e], mean2), rstd2), w[j * N / 2 + e], b[j * N / 2 + e]);
                reinterpret_cast<uint4*>(yr)[j * THREADS + at] = f2_piece<T>(f);
            }
        if (at == 0) {
            if (a.stats) a.stats[r] = make_float2(mean, rstd);
            if (a.q) a.q_scale[r] = scale.scale;
        }
    }
    if (failed) ring.drain(i, min(mine, i + a.stages));
}

// What the gradient takes its normalised rows from: x, or 8-bit rows with scales.
struct LnGrad {
    int64_t rows, cols, lddy, ldx, lddx;
    const void* dy;
    const void* x;          // or
    const int8_t* q;
    const float* q_scale;
    const float2* stats;
    const float* weight;
    void* dx;
    float* lines;           // [CTAs][2][cols]: sums of dy xh and of dy
    int columns;            // whether these are wanted
    int stages, bytes;      // of the ring
    s2v_device_status* status;
};

template <typename T, bool VEC, int NV, int THREADS, bool FROM8>
__global__ void __launch_bounds__(THREADS < LN_CTA ? LN_CTA : THREADS) layer_norm_grad_kernel(const LnGrad a)
{
    using P = ln_piece<T, VEC>;
    constexpr int N = P::N, CTA = THREADS < LN_CTA ? LN_CTA : THREADS, WARPS = THREADS / 32, GROUPS = CTA / THREADS;
    __shared__ float2 part[WARPS > 1 ? 2 * WARPS : 1];
    extern __shared__ float ln_lines[];   // GROUPS > 1: a line of sums at a time
    const int at = threadIdx.x % THREADS;
    const int pieces = (int)(a.cols / N);
    float sum_w[NV * N] = {}, sum_b[NV * N] = {};
    int turn = 0;
    for (int64_t first = (int64_t)blockIdx.x * GROUPS; first < a.rows; first += (int64_t)gridDim.x * GROUPS, turn ^= 1) {
        const int64_t own = first + threadIdx.x / THREADS, r = min(own, a.rows - 1);
        const bool mine = own < a.rows;
        const T* const dyr = static_cast<const T*>(a.dy) + r * a.lddy;
        const float2 st = a.stats[r];
        const float s = FROM8 ? a.q_scale[r] : 1.0f;
        typename P::raw dv[NV];
        typename std::conditional<FROM8, typename P::raw8, typename P::raw>::type xv[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < pieces) {
                dv[j] = P::load(dyr, j * THREADS + at);
                if constexpr (FROM8) xv[j] = P::load8(a.q + r * a.ldx, j * THREADS + at);
                else xv[j] = P::load(static_cast<const T*>(a.x) + r * a.ldx, j * THREADS + at);
            }
        const auto normalised = [&](int j, float* h) {
            if constexpr (FROM8) P::unpack8(xv[j], h);
            else P::unpack(xv[j], h);
#pragma unroll
            for (int e = 0; e < N; ++e) h[e] = FROM8 ? fmaf(h[e], s, -st.x) * st.y : (h[e] - st.x) * st.y;
        };
        float g0 = 0.0f, g1 = 0.0f;   // sums of g = dy w and of g xh
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < pieces) {
                float d[N], h[N], w[N];
                P::unpack(dv[j], d);
                normalised(j, h);
                P::columns(a.weight, j * THREADS + at, 1.0f, w);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float g = d[e] * w[e];
                    g0 += g;
                    g1 = fmaf(g, h[e], g1);
                    if (mine) sum_w[j * N + e] = fmaf(d[e], h[e], sum_w[j * N + e]), sum_b[j * N + e] += d[e];
                }
            }
#pragma unroll
        for (int o = (THREADS < 32 ? THREADS : 32) / 2; o; o >>= 1) g0 += __shfl_xor_sync(0xffffffffu, g0, o), g1 += __shfl_xor_sync(0xffffffffu, g1, o);
        if constexpr (WARPS > 1) {
            if ((at & 31) == 0) part[turn * WARPS + (at >> 5)] = make_float2(g0, g1);
            __syncthreads();
            g0 = g1 = 0.0f;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) g0 += part[turn * WARPS + i].x, g1 += part[turn * WARPS + i].y;
        }
        if (!mine) continue;
        const float inv = 1.0f / (float)a.cols, m0 = g0 * inv, m1 = g1 * inv;
        T* const dxr = static_cast<T*>(a.dx) + r * a.lddx;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < pieces) {
                float d[N], h[N], w[N];
                P::unpack(dv[j], d);
                normalised(j, h);
                P::columns(a.weight, j * THREADS + at, 1.0f, w);
#pragma unroll
                for (int e = 0; e < N; ++e) d[e] = st.y * (fmaf(d[e], w[e], -m0) - h[e] * m1);
                P::store(dxr, j * THREADS + at, d);
            }
    }
    if (!a.columns) return;
    float* const line = a.lines + (int64_t)blockIdx.x * 2 * a.cols;
    if constexpr (GROUPS == 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + at < pieces)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    line[(int64_t)(j * THREADS + at) * N + e] = sum_w[j * N + e];
                    line[a.cols + (int64_t)(j * THREADS + at) * N + e] = sum_b[j * N + e];
                }
    } else {   // groups of a warp by shuffles, warps through shared memory
#pragma unroll
        for (int i = 0; i < NV * N; ++i)
#pragma unroll
            for (int o = THREADS; o < 32; o <<= 1) sum_w[i] += __shfl_xor_sync(0xffffffffu, sum_w[i], o), sum_b[i] += __shfl_xor_sync(0xffffffffu, sum_b[i], o);
        constexpr int LINE = NV * N * THREADS, CW = CTA / 32;
        for (int half = 0; half < 2; ++half) {
            if ((threadIdx.x & 31) < THREADS) {
#pragma unroll
                for (int i = 0; i < NV * N; ++i) ln_lines[(threadIdx.x >> 5) * LINE + (i / N * THREADS + at) * N + i % N] = half ? sum_b[i] : sum_w[i];
            }
            __syncthreads();
            for (int c = threadIdx.x; c < a.cols; c += CTA) {
                float t = 0.0f;
                for (int w = 0; w < CW; ++w) t += ln_lines[w * LINE + c];
                line[half * a.cols + c] = t;
            }
            __syncthreads();
        }
    }
}

// The same through the ring, R rows a turn of a CTA: a stage holds a row's dy and, behind it, x or the 8-bit row.  With the rows' raw numbers and the weight in
// registers a number is read from shared memory once, and R rows share a barrier.  (8192 x 8192 bf16, 83 us: the instructions, 27 a number, half of them what a
// row costs a thread; 32 numbers a thread of two CTAs an SM, with dy and 8-bit rows read twice and the weight twice a row through L1 105, with g = dy w kept in
// registers, some of them spilled, 119; before the ring was kept count of without divisions 97.)
template <typename T, int NV, int R, int THREADS, int CTAS, bool FROM8> __global__ void __launch_bounds__(THREADS, CTAS) layer_norm_grad_ring_kernel(const LnGrad a)
{
    using P = ln_piece<T, true>;
    using raw_x = typename std::conditional<FROM8, typename P::raw8, uint4>::type;
    constexpr int N = P::N, WARPS = THREADS / 32;
    __shared__ float2 part[2][R][WARPS];
    extern __shared__ unsigned char ln_raw[];
    const ln_ring ring(ln_raw, a.stages, a.bytes);
    const int at = threadIdx.x, pieces = (int)(a.cols / N), row_bytes = (int)(a.cols * (int64_t)sizeof(T)), x_bytes = FROM8 ? (int)a.cols : row_bytes;
    const int mine = (int)((a.rows - blockIdx.x + gridDim.x - 1) / gridDim.x);   // rows of this CTA
    const auto fetch = [&](int i, int stage) {
        if (i < mine) {
            const int64_t r = (int64_t)blockIdx.x + (int64_t)i * gridDim.x;
            mbar_expect(ring.full + 8 * stage, (uint32_t)(row_bytes + x_bytes));
            ring.copy(stage, 0, static_cast<const T*>(a.dy) + r * a.lddy, row_bytes);
            if constexpr (FROM8) ring.copy(stage, row_bytes, a.q + r * a.ldx, x_bytes);
            else ring.copy(stage, row_bytes, static_cast<const T*>(a.x) + r * a.ldx, x_bytes);
        }
    };
    if (at == 0)
        for (int i = 0; i < a.stages; ++i) fetch(i, i);
    uint64_t w[NV * N / 2], sum_w[NV * N / 2] = {}, sum_b[NV * N / 2] = {};   // (zeros)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        float u[N];
#pragma unroll
        for (int e = 0; e < N; ++e) u[e] = 0.0f;
        if (j * THREADS + at < pieces) P::columns(a.weight, j * THREADS + at, 1.0f, u);
#pragma unroll
        for (int e = 0; e < N / 2; ++e) w[j * N / 2 + e] = f2_of(u[2 * e], u[2 * e + 1]);
    }
    const float inv = 1.0f / (float)a.cols;
    int i = 0, stage = 0;
    uint32_t phase = 0;
    bool failed = false;
    float2 next_st[R];
    float next_s[R];
    const auto ask = [&](int from) {   // the rows' numbers, a turn ahead
#pragma unroll
        for (int u = 0; u < R; ++u)
            if (from + u < mine) {
                const int64_t r = (int64_t)blockIdx.x + (int64_t)(from + u) * gridDim.x;
                next_st[u] = a.stats[r], next_s[u] = FROM8 ? a.q_scale[r] : 1.0f;
            }
    };
    ask(0);
    for (; i < mine; i += R) {
        float2 st[R];
        float s[R];
#pragma unroll
        for (int u = 0; u < R; ++u) st[u] = next_st[u], s[u] = next_s[u];
        ask(i + R);
        uint4 dv[R][NV];
        raw_x xv[R][NV];
        // normalised numbers of a piece
        const auto normalise = [&](int u, const raw_x& v, uint64_t* h) {
            const uint64_t mean2 = f2_of(-st[u].x, -st[u].x), rstd2 = f2_of(st[u].y, st[u].y), s2 = f2_of(s[u], s[u]);
            if constexpr (!FROM8) f2_unpack<T>(v, h);
            else if constexpr (N == 8) f2_unpack8(v.x, h), f2_unpack8(v.y, h + 2);
            else f2_unpack8(v, h);
#pragma unroll
            for (int e = 0; e < N / 2; ++e) h[e] = f2_mul(FROM8 ? f2_fma(h[e], s2, mean2) : f2_add(h[e], mean2), rstd2);
        };
        bool ok = true;
        float g0[R], g1[R];
        int at_stage[R];
#pragma unroll
        for (int u = 0; u < R; ++u) {
            uint64_t s0 = 0, s1 = 0;
            at_stage[u] = stage;
            if (i + u < mine) {
                ok = ok && ring.wait(stage, phase, a.status);
                const unsigned char* const from = ring.at + stage * a.bytes;
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (j * THREADS + at < pieces) {
                        dv[u][j] = reinterpret_cast<const uint4*>(from)[j * THREADS + at];
                        xv[u][j] = reinterpret_cast<const raw_x*>(from + row_bytes)[j * THREADS + at];
                        uint64_t d[N / 2], h[N / 2];
                        f2_unpack<T>(dv[u][j], d);
                        normalise(u, xv[u][j], h);
#pragma unroll
                        for (int e = 0; e < N / 2; ++e) {
                            const int c = j * N / 2 + e;
                            const uint64_t g = f2_mul(d[e], w[c]);
                            s1 = f2_fma(g, h[e], s1), s0 = f2_fma(d[e], w[c], s0);
                            sum_w[c] = f2_fma(d[e], h[e], sum_w[c]), sum_b[c] = f2_add(sum_b[c], d[e]);
                        }
                    }
            }
            if (++stage == a.stages) stage = 0, phase ^= 1;
            g0[u] = f2_sum(s0), g1[u] = f2_sum(s1);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1)
#pragma unroll
            for (int u = 0; u < R; ++u) g0[u] += __shfl_xor_sync(0xffffffffu, g0[u], o), g1[u] += __shfl_xor_sync(0xffffffffu, g1[u], o);
        const int turn = i / R & 1;
        if ((at & 31) == 0) {
#pragma unroll
            for (int u = 0; u < R; ++u) part[turn][u][at >> 5] = make_float2(g0[u], g1[u]);
        }
        if (__syncthreads_or(!ok)) {
            failed = true;
            break;
        }
        if (at == 0) {   // (the rows are in registers)
#pragma unroll
            for (int u = 0; u < R; ++u) fetch(i + u + a.stages, at_stage[u]);
        }
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const float2 p = part[turn][u][at & (WARPS - 1)];
            g0[u] = ln_lanes_sum<WARPS>(p.x), g1[u] = ln_lanes_sum<WARPS>(p.y);
        }
#pragma unroll
        for (int u = 0; u < R; ++u) {
            if (i + u >= mine) break;
            const uint64_t m0 = f2_of(-g0[u] * inv, -g0[u] * inv), m1 = f2_of(-g1[u] * inv, -g1[u] * inv), rstd2 = f2_of(st[u].y, st[u].y);
            uint4* const dxr = reinterpret_cast<uint4*>(static_cast<T*>(a.dx) + ((int64_t)blockIdx.x + (int64_t)(i + u) * gridDim.x) * a.lddx);
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (j * THREADS + at < pieces) {
                    uint64_t d[N / 2], h[N / 2];
                    f2_unpack<T>(dv[u][j], d);
                    normalise(u, xv[u][j], h);
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) d[e] = f2_mul(rstd2, f2_fma(h[e], m1, f2_fma(d[e], w[j * N / 2 + e], m0)));
                    dxr[j * THREADS + at] = f2_piece<T>(d);
                }
        }
    }
    if (failed) {
        ring.drain(i, min(mine, i + a.stages));
        return;
    }
    if (!a.columns) return;
    float* const line = a.lines + (int64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if (j * THREADS + at < pieces)
#pragma unroll
            for (int e = 0; e < N / 2; e += 2) {
                const int c = (j * THREADS + at) * N + 2 * e;
                *reinterpret_cast<ulonglong2*>(line + c) = make_ulonglong2(sum_w[j * N / 2 + e], sum_w[j * N / 2 + e + 1]);
                *reinterpret_cast<ulonglong2*>(line + a.cols + c) = make_ulonglong2(sum_b[j * N / 2 + e], sum_b[j * N / 2 + e + 1]);
            }
}

// Rows longer than a CTA's registers: read twice, and a second kernel for the columns' sums.
template <typename T, bool FROM8> __global__ void __launch_bounds__(512) layer_norm_grad_long_kernel(const LnGrad a)
{
    __shared__ float2 part[2 * 16];
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
        const T* const dyr = static_cast<const T*>(a.dy) + r * a.lddy;
        T* const dxr = static_cast<T*>(a.dx) + r * a.lddx;
        const float2 st = a.stats[r];
        const float s = FROM8 ? a.q_scale[r] : 1.0f;
        const auto normalised = [&](int64_t c) { return FROM8 ? fmaf((float)a.q[r * a.ldx + c], s, -st.x) * st.y : (to_f32(static_cast<const T*>(a.x)[r * a.ldx + c]) - st.x) * st.y; };
        float g0 = 0.0f, g1 = 0.0f;
        for (int64_t c = threadIdx.x; c < a.cols; c += 512) {
            const float g = to_f32(dyr[c]) * (a.weight ? __ldg(a.weight + c) : 1.0f);
            g0 += g;
            g1 = fmaf(g, normalised(c), g1);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) g0 += __shfl_xor_sync(0xffffffffu, g0, o), g1 += __shfl_xor_sync(0xffffffffu, g1, o);
        if ((threadIdx.x & 31) == 0) part[turn * 16 + (threadIdx.x >> 5)] = make_float2(g0, g1);
        __syncthreads();
        g0 = g1 = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) g0 += part[turn * 16 + i].x, g1 += part[turn * 16 + i].y;
        const float m0 = g0 / (float)a.cols, m1 = g1 / (float)a.cols;
        for (int64_t c = threadIdx.x; c < a.cols; c += 512)
            dxr[c] = from_f32<T>(st.y * (fmaf(to_f32(dyr[c]), a.weight ? __ldg(a.weight + c) : 1.0f, -m0) - normalised(c) * m1));
    }
}
// a column a thread, a share of the rows a CTA
template <typename T, bool FROM8> __global__ void __launch_bounds__(LN_CTA) layer_norm_columns_kernel(const LnGrad a, int64_t share)
{
    const int64_t c = (int64_t)blockIdx.x * LN_CTA + threadIdx.x, from = blockIdx.y * share, to = min(a.rows, from + share);
    if (c >= a.cols) return;
    float w = 0.0f, b = 0.0f;
    for (int64_t r = from; r < to; ++r) {
        const float d = to_f32(static_cast<const T*>(a.dy)[r * a.lddy + c]);
        const float2 st = a.stats[r];
        const float h = FROM8 ? fmaf((float)a.q[r * a.ldx + c], a.q_scale[r], -st.x) * st.y : (to_f32(static_cast<const T*>(a.x)[r * a.ldx + c]) - st.x) * st.y;
        w = fmaf(d, h, w);
        b += d;
    }
    float* const line = a.lines + (int64_t)blockIdx.y * 2 * a.cols;
    line[c] = w, line[a.cols + c] = b;
}
// The lines of the gradient's CTAs, added in a fixed order: V columns a thread, LANES threads side by side, the others a share of the lines each.
template <int V, int LANES> __global__ void __launch_bounds__(LN_CTA) layer_norm_lines_kernel(int lines, int64_t cols, const float* __restrict__ from, float* __restrict__ dweight, float* __restrict__ dbias)
{
    constexpr int SHARES = LN_CTA / LANES;
    __shared__ float part[SHARES][LANES * V];
    const int at = threadIdx.x % LANES, g = threadIdx.x / LANES;
    const int64_t c = ((int64_t)blockIdx.x * LANES + at) * V;
    float t[V] = {};
    if (c < 2 * cols) {
#pragma unroll 8
        for (int l = g; l < lines; l += SHARES) {
            if constexpr (V == 4) {
                const float4 f = __ldcs(reinterpret_cast<const float4*>(from + (int64_t)l * 2 * cols + c));
                t[0] += f.x, t[1] += f.y, t[2] += f.z, t[3] += f.w;
            } else t[0] += __ldcs(from + (int64_t)l * 2 * cols + c);
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) part[g][at * V + e] = t[e];
    __syncthreads();
    if (threadIdx.x >= LANES * V) return;
    const int64_t k = (int64_t)blockIdx.x * LANES * V + threadIdx.x;
    float s = 0.0f;
#pragma unroll 8
    for (int i = 0; i < SHARES; ++i) s += part[i][threadIdx.x];
    if (k < cols) {
        if (dweight) dweight[k] = s;
    } else if (k < 2 * cols && dbias) dbias[k - cols] = s;
}

// Stages of a ring for `ctas` CTAs on an SM: what fits, LN_STAGES at most.
constexpr int LN_RING_ROW = 65536;   // bytes of a stage
constexpr size_t LN_RING_SHARED = 222 * 1024, LN_RING_LESS = 168 * 1024;   // of an SM; where the smaller has room for two stages, the rest is L1's
template <typename K, typename A> int ln_ring_stages(s2v_ctx* ctx, K kernel, A& a, int ctas)
{
    const size_t fixed = ln_ring::shared(0, 0) + 1024 + 512;   // (what a CTA takes besides, and the kernel's own)
    const auto stages = [&](size_t shared) { return (int)((shared / ctas - fixed) / a.bytes); };
    a.stages = stages(LN_RING_LESS) >= 2 ? stages(LN_RING_LESS) : stages(LN_RING_SHARED);
    a.stages = a.stages < LN_STAGES ? a.stages : LN_STAGES;
    S2V_CUDA_OK(ctx, s2v_allow_shared(kernel, LN_RING_SHARED));
    return S2V_OK;
}

template <typename T, bool VEC>
int ln_launch(s2v_ctx* ctx, cudaStream_t st, int64_t rows, int64_t cols, const T* x, int64_t ldx, const float* weight, const float* bias, float eps, T* y, int64_t ldy,
              float2* stats, int8_t* q, int64_t ldq, float* q_scale)
{
    const int64_t pieces = cols / ln_piece<T, VEC>::N;
    const auto go = [&](auto kernel, int threads) {
        const int per = threads < LN_CTA ? LN_CTA / threads : 1;
        const int64_t blocks = (rows + per - 1) / per, cap = (int64_t)1 << 20;
        kernel<<<(unsigned)(blocks < cap ? blocks : cap), threads < LN_CTA ? LN_CTA : threads, 0, st>>>(rows, cols, x, ldx, weight, bias, eps, y, ldy, stats, q, ldq, q_scale);
        S2V_CHECK_LAUNCH(ctx, "layer_norm_kernel");
        return (int)S2V_OK;
    };
    if constexpr (VEC) {
        if (pieces > 128 && cols <= 16384 && rows <= INT32_MAX) {
            LnNorm a{rows, cols, ldx, ldy, ldq, x, weight, bias, eps, y, stats, q, q_scale, 0, (int)((pieces * 16 + 127) / 128 * 128), ctx->dstatus_dev};
            const auto ring = [&](auto kernel, int threads, int ctas) {
                const int rc = ln_ring_stages(ctx, kernel, a, ctas);
                if (rc != S2V_OK) return rc;
                const int64_t most = (int64_t)ctas * ctx->sm_count;
                kernel<<<(unsigned)(rows < most ? rows : most), threads, ln_ring::shared(a.stages, a.bytes), st>>>(a);
                S2V_CHECK_LAUNCH(ctx, "layer_norm_ring_kernel");
                return (int)S2V_OK;
            };
            constexpr int N = ln_piece<T, true>::N;
            if (cols <= 2048) return ring(layer_norm_ring_kernel<T, 32 / N, 64, 8>, 64, 8);
            if (cols <= 4096) return ring(layer_norm_ring_kernel<T, 32 / N, 128, 4>, 128, 4);
            if (cols <= 8192) return ring(layer_norm_ring_kernel<T, 32 / N, 256, 2>, 256, 2);
            if (cols <= 16384) return ring(layer_norm_ring_kernel<T, 32 / N, 512, 1>, 512, 1);
        }
    }
    if (pieces <= 8) return go(layer_norm_kernel<T, VEC, 1, 8>, 8);
    if (pieces <= 32) return go(layer_norm_kernel<T, VEC, 4, 8>, 8);
    if (pieces <= 128) return go(layer_norm_kernel<T, VEC, 4, 32>, 32);
    if constexpr (!VEC) {   // (rows in pieces of 16 bytes go through the ring; no memory holds more rows than it takes)
        if (pieces <= 512) return go(layer_norm_kernel<T, VEC, 2, 256>, 256);
        if (pieces <= 1024) return go(layer_norm_kernel<T, VEC, 4, 256>, 256);
    }
    return go(layer_norm_kernel<T, VEC, 8, 256>, 256);
}

int ln_ctas(const s2v_ctx* ctx, int64_t rows, int per)
{
    const int64_t turns = (rows + per - 1) / per, most = 4 * (int64_t)ctx->sm_count;
    return (int)(turns < most ? turns : most < LN_MAX_LINES ? most : LN_MAX_LINES);
}

template <typename T, bool FROM8> int ln_grad_launch(s2v_ctx* ctx, cudaStream_t st, const LnGrad& a, bool vec, float* dweight, float* dbias)
{
    int lines = 0;
    const auto go = [&](auto kernel, int threads, int line) {
        const int per = threads < LN_CTA ? LN_CTA / threads : 1;
        lines = ln_ctas(ctx, a.rows, per);
        kernel<<<lines, threads < LN_CTA ? LN_CTA : threads, threads < LN_CTA ? LN_CTA / 32 * line * sizeof(float) : 0, st>>>(a);
        S2V_CHECK_LAUNCH(ctx, "layer_norm_grad_kernel");
        return (int)S2V_OK;
    };
    const auto ring = [&](auto kernel, int threads, int ctas) {
        LnGrad r = a;
        r.bytes = (int)((a.cols * (int64_t)(sizeof(T) + (FROM8 ? 1 : sizeof(T))) + 127) / 128 * 128), r.status = ctx->dstatus_dev;
        const int rc = ln_ring_stages(ctx, kernel, r, ctas);
        if (rc != S2V_OK) return rc;
        const int64_t most = (int64_t)ctas * ctx->sm_count;
        lines = (int)(a.rows < most ? a.rows : most);
        kernel<<<lines, threads, ln_ring::shared(r.stages, r.bytes), st>>>(r);
        S2V_CHECK_LAUNCH(ctx, "layer_norm_grad_ring_kernel");
        return (int)S2V_OK;
    };
    const auto by_size = [&](auto vector) {
        constexpr bool VEC = decltype(vector)::value;
        constexpr int N = ln_piece<T, VEC>::N;
        const int64_t pieces = a.cols / N;
        if constexpr (VEC) {
            // (at least two rows of a CTA in the ring; the 8-bit rows on 16-byte boundaries too)
            const bool whole = !FROM8 || (a.cols % 16 == 0 && s2v_aligned16(a.q) && (a.rows <= 1 || a.ldx % 16 == 0));
            if (pieces > 128 && whole && a.rows <= INT32_MAX && a.cols * (int64_t)(sizeof(T) + (FROM8 ? 1 : sizeof(T))) <= LN_RING_ROW) {
                if (pieces <= 256) return ring(layer_norm_grad_ring_kernel<T, 2, 2, 128, 4, FROM8>, 128, 4);
                if (pieces <= 512) return ring(layer_norm_grad_ring_kernel<T, 2, 2, 256, 2, FROM8>, 256, 2);
                if (pieces <= 1024) return ring(layer_norm_grad_ring_kernel<T, 2, 2, 512, 1, FROM8>, 512, 1);
                if constexpr (N == 4) {
                    if (pieces <= 2048) return ring(layer_norm_grad_ring_kernel<T, 4, 1, 512, 1, FROM8>, 512, 1);
                }
            }
        }
        if (pieces <= 8) return go(layer_norm_grad_kernel<T, VEC, 1, 8, FROM8>, 8, 8 * N);
        if (pieces <= 32) return go(layer_norm_grad_kernel<T, VEC, 4, 8, FROM8>, 8, 32 * N);
        if (pieces <= 128) return go(layer_norm_grad_kernel<T, VEC, 4, 32, FROM8>, 32, 128 * N);
        constexpr bool RING = VEC && !FROM8;   // rows of x in pieces of 16 bytes go through the ring, up to its limits; 8-bit rows may lie at other places
        if constexpr (!RING) {
            if (pieces <= 512) return go(layer_norm_grad_kernel<T, VEC, 2, 256, FROM8>, 256, 0);
            if (pieces <= 1024) return go(layer_norm_grad_kernel<T, VEC, 2, 512, FROM8>, 512, 0);
        }
        if constexpr (!RING || N == 8) {
            if (pieces <= 2048) return go(layer_norm_grad_kernel<T, VEC, 4, 512, FROM8>, 512, 0);
        }
        if constexpr (N < 8) {
            if (pieces <= 4096) return go(layer_norm_grad_kernel<T, VEC, 8, 512, FROM8>, 512, 0);
        }
        if (a.columns) {   // (first: dx may lie over dy)
            const int64_t blocks = (a.cols + LN_CTA - 1) / LN_CTA;
            if (blocks > INT32_MAX) return s2v_fail(ctx, S2V_ERR_UNSUPPORTED, "layer_norm_grad: too many columns");
            lines = ln_ctas(ctx, a.rows, 16);
            const int64_t share = (a.rows + lines - 1) / lines;
            lines = (int)((a.rows + share - 1) / share);
            layer_norm_columns_kernel<T, FROM8><<<dim3((unsigned)blocks, lines), LN_CTA, 0, st>>>(a, share);
            S2V_CHECK_LAUNCH(ctx, "layer_norm_columns_kernel");
        }
        const int64_t cap = (int64_t)1 << 20;
        layer_norm_grad_long_kernel<T, FROM8><<<(unsigned)(a.rows < cap ? a.rows : cap), 512, 0, st>>>(a);
        S2V_CHECK_LAUNCH(ctx, "layer_norm_grad_long_kernel");
        return (int)S2V_OK;
    };
    const int rc = vec ? by_size(std::true_type()) : by_size(std::false_type());
    if (rc != S2V_OK || !a.columns) return rc;
    // (eight threads side by side where columns are few: 592 lines of 2 x 128 columns by two CTAs of 32 took 22 us)
    const auto add = [&](auto kernel, int64_t per) { kernel<<<(unsigned)((2 * a.cols + per - 1) / per), LN_CTA, 0, st>>>(lines, a.cols, a.lines, dweight, dbias); };
    if (a.cols % 2 == 0) a.cols >= 4096 ? add(layer_norm_lines_kernel<4, 16>, 64) : add(layer_norm_lines_kernel<4, 4>, 16);
    else a.cols >= 4096 ? add(layer_norm_lines_kernel<1, 32>, 32) : add(layer_norm_lines_kernel<1, 8>, 8);
    S2V_CHECK_LAUNCH(ctx, "layer_norm_lines_kernel");
    return S2V_OK;
}

// Whether every row of a matrix lies on a boundary of `bytes`.
bool rows_aligned(const void* p, int64_t rows, int64_t ld, int64_t es, int64_t bytes)
{
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (rows <= 1 || ld * es % bytes == 0);
}

}  // namespace

extern "C" {

int s2v_layer_norm(s2v_ctx* ctx, s2v_stream stream, int64_t rows, int64_t cols, int x_type, const void* x, int64_t ldx, const float* weight, const float* bias, float eps,
                   void* y, int64_t ldy, float* stats, int8_t* q, int64_t ldq, float* q_scale)
{
    S2V_ENTER(ctx);
    const auto bad = [&](int status, const char* what) { return s2v_fail(ctx, status, std::string("layer_norm: ") + what); };
    if (rows < 0 || cols < 1) return bad(S2V_ERR_INVALID_ARG, "negative size or no columns");
    if (!s2v_dtype_ok(x_type)) return bad(S2V_ERR_INVALID_ARG, "unknown element type");
    if (!(eps >= 0.0f) || eps > 1e30f) return bad(S2V_ERR_INVALID_ARG, "eps outside 0 to 1e30");
    if (rows == 0) return S2V_OK;
    if (cols > INT32_MAX) return bad(S2V_ERR_UNSUPPORTED, "more than 2^31 - 1 columns");
    if (!x || !y || (q == nullptr) != (q_scale == nullptr)) return bad(S2V_ERR_INVALID_ARG, "NULL pointer");
    if (rows > 1 && (ldx < cols || ldy < cols || (q && ldq < cols))) return bad(S2V_ERR_INVALID_ARG, "leading dimension below the number of columns");
    if (x == y && rows > 1 && ldx != ldy) return bad(S2V_ERR_INVALID_ARG, "in place with another leading dimension");
    const int64_t es = (int64_t)s2v_dtype_bytes(x_type);
    if (reinterpret_cast<uintptr_t>(x) % es || reinterpret_cast<uintptr_t>(y) % es || reinterpret_cast<uintptr_t>(stats) % 8 || !s2v_aligned4(weight, bias, q_scale))
        return bad(S2V_ERR_INVALID_ARG, "misaligned pointer");
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    const bool vec = cols % (16 / es) == 0 && rows_aligned(x, rows, ldx, es, 16) && rows_aligned(y, rows, ldy, es, 16);
    return s2v_by_dtype(x_type, [&](auto type) {
        using T = decltype(type);
        const auto go = [&](auto vector) {
            return ln_launch<T, decltype(vector)::value>(ctx, st, rows, cols, static_cast<const T*>(x), ldx, weight, bias, eps, static_cast<T*>(y), ldy,
                                                         reinterpret_cast<float2*>(stats), q, ldq, q_scale);
        };
        return vec ? go(std::true_type()) : go(std::false_type());
    });
}

size_t s2v_layer_norm_grad_workspace_bytes(int64_t rows, int64_t cols)
{
    if (rows <= 0 || cols <= 0 || cols > INT32_MAX) return 0;
    return (size_t)(rows < LN_MAX_LINES ? rows : LN_MAX_LINES) * 2 * (size_t)cols * sizeof(float);
}

int s2v_layer_norm_grad(s2v_ctx* ctx, s2v_stream stream, int64_t rows, int64_t cols, int type, const void* dy, int64_t lddy, const void* x, int64_t ldx, const int8_t* q,
                        int64_t ldq, const float* q_scale, const float* stats, const float* weight, void* workspace, size_t workspace_bytes, void* dx, int64_t lddx,
                        float* dweight, float* dbias)
{
    S2V_ENTER(ctx);
    const auto bad = [&](int status, const char* what) { return s2v_fail(ctx, status, std::string("layer_norm_grad: ") + what); };
    if (rows < 0 || cols < 1) return bad(S2V_ERR_INVALID_ARG, "negative size or no columns");
    if (!s2v_dtype_ok(type)) return bad(S2V_ERR_INVALID_ARG, "unknown element type");
    if (cols > INT32_MAX) return bad(S2V_ERR_UNSUPPORTED, "more than 2^31 - 1 columns");
    if (!s2v_aligned4(weight, q_scale, dweight, dbias) || reinterpret_cast<uintptr_t>(stats) % 8) return bad(S2V_ERR_INVALID_ARG, "misaligned pointer");
    cudaStream_t st = s2v_pick_stream(ctx, stream);
    if (rows == 0) {   // empty sums
        if (dweight) S2V_CUDA_OK(ctx, cudaMemsetAsync(dweight, 0, (size_t)cols * sizeof(float), st));
        if (dbias) S2V_CUDA_OK(ctx, cudaMemsetAsync(dbias, 0, (size_t)cols * sizeof(float), st));
        return S2V_OK;
    }
    if (!dy || !dx || !stats) return bad(S2V_ERR_INVALID_ARG, "NULL pointer");
    if ((x == nullptr) == (q == nullptr) || (q == nullptr) != (q_scale == nullptr)) return bad(S2V_ERR_INVALID_ARG, "takes x, or q and its scales");
    if (rows > 1 && (lddy < cols || lddx < cols || (x ? ldx : ldq) < cols)) return bad(S2V_ERR_INVALID_ARG, "leading dimension below the number of columns");
    if (dx == dy && rows > 1 && lddx != lddy) return bad(S2V_ERR_INVALID_ARG, "in place with another leading dimension");
    const int64_t es = (int64_t)s2v_dtype_bytes(type);
    if (reinterpret_cast<uintptr_t>(dy) % es || reinterpret_cast<uintptr_t>(x) % es || reinterpret_cast<uintptr_t>(dx) % es) return bad(S2V_ERR_INVALID_ARG, "misaligned pointer");
    if (dweight || dbias) {
        if (!workspace || workspace_bytes < s2v_layer_norm_grad_workspace_bytes(rows, cols)) return bad(S2V_ERR_WORKSPACE, "workspace too small");
        if (!s2v_aligned16(workspace)) return bad(S2V_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
    }
    LnGrad a{rows, cols, lddy, x ? ldx : ldq, lddx, dy, x, q, q_scale, reinterpret_cast<const float2*>(stats), weight, dx, static_cast<float*>(workspace), dweight || dbias, 0, 0, nullptr};
    const int64_t n = 16 / es;
    const bool vec = cols % n == 0 && rows_aligned(dy, rows, lddy, es, 16) && rows_aligned(dx, rows, lddx, es, 16) &&
                     (x ? rows_aligned(x, rows, ldx, es, 16) : rows_aligned(q, rows, ldq, 1, n));
    return s2v_by_dtype(type, [&](auto t) {
        using T = decltype(t);
        return q ? ln_grad_launch<T, true>(ctx, st, a, vec, dweight, dbias) : ln_grad_launch<T, false>(ctx, st, a, vec, dweight, dbias);
    });
}

}  // extern "C"
