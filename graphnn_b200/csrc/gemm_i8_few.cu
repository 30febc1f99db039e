// Products with few tokens, where reading the weights once is everything: a kernel without matrix instructions for one or two tokens (which also
// quantises them on the way), and one that splits k among the CTAs of a cluster for outputs of few tiles.
#include <cmath>

#include "gemm_i8.cuh"
#include "quantize.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace
{

// ---------------------------------------------------------------- one or two tokens
// A warp per weight row: 32 lanes read 512 bytes of it at a time, eight such loads on their way at once, before the tokens are even looked at.  The
// tokens lie in shared memory as 8-bit integers, quantised by every CTA for itself (they are few; a launch in front would take as long as this
// one).  dp4a adds up four products; a lane's sums are joined at the end.
constexpr int GV_THREADS = 256, GV_WARPS = GV_THREADS / 32, GV_AHEAD = 8;
constexpr uint32_t GV_SMEM = 64 << 10;   // bytes of tokens, at most

struct GvArgs {
    int64_t n, k, ldx, ldw, ldy;
    int m, kp;             // kp: k rounded up to 16
    const void* x;
    const float* x_scale;  // 8-bit x
    const int8_t* W;
    const float* w_scale;
    const float* bias;
    int relu;
    void* y;
};

template <int M> __device__ __forceinline__ void gv_add(int (&acc)[M], const uint4& w, const int8_t* xs, int kp, int off)
{
#pragma unroll
    for (int t = 0; t < M; ++t) {
        const uint4 x = *reinterpret_cast<const uint4*>(xs + t * kp + off);
        int s = acc[t];
        s = __dp4a((int)w.x, (int)x.x, s);
        s = __dp4a((int)w.y, (int)x.y, s);
        s = __dp4a((int)w.z, (int)x.z, s);
        acc[t] = __dp4a((int)w.w, (int)x.w, s);
    }
}

template <typename TX, typename TY, int M>
__global__ void __launch_bounds__(GV_THREADS, 4) gemv_i8_kernel(const GvArgs a)
{
    extern __shared__ __align__(16) int8_t xs[];   // [M][kp]
    __shared__ float sx[M];
    __shared__ uint32_t part[GV_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t groups = (a.n + GV_WARPS - 1) / GV_WARPS;
    const int kp = a.kp, chunks = ((int)a.k + 511) / 512;
    uint4 w[GV_AHEAD];
    const int8_t* wr;
    const int k16 = (int)a.k & ~15, rest = (int)a.k & 15;   // whole pieces; the last bytes are multiplied one by one (a matrix may end with its last row)
    const auto row_of = [&](int64_t g) { return min(g * GV_WARPS + warp, a.n - 1); };   // (rows behind the last are computed as the last and not written)
    const auto fetch = [&](int c0) {
#pragma unroll
        for (int c = 0; c < GV_AHEAD; ++c)
            if (const int off = (c0 + c) * 512 + lane * 16; off < k16) w[c] = __ldcs(reinterpret_cast<const uint4*>(wr + off));
    };
    wr = a.W + row_of(blockIdx.x) * a.ldw;
    fetch(0);
    // the tokens: GV_WARPS / M warps each
    if constexpr (std::is_same<TX, int8_t>::value) {
        for (int t = 0; t < M; ++t) {
            const int8_t* const xr = static_cast<const int8_t*>(a.x) + min(t, a.m - 1) * a.ldx;
            for (int o = threadIdx.x * 16; o < k16; o += GV_THREADS * 16) *reinterpret_cast<uint4*>(xs + t * kp + o) = __ldg(reinterpret_cast<const uint4*>(xr + o));
            if (threadIdx.x < rest) xs[t * kp + k16 + threadIdx.x] = xr[k16 + threadIdx.x];
        }
        if (threadIdx.x < M) sx[threadIdx.x] = threadIdx.x < a.m ? a.x_scale[threadIdx.x] : 0.0f;
    } else {
        constexpr int EACH = GV_THREADS / M, N = PIECE<TX>;
        const int t = threadIdx.x / EACH, at = threadIdx.x % EACH;
        const TX* const xr = static_cast<const TX*>(a.x) + min(t, a.m - 1) * a.ldx;
        const row_pieces<TX> row(xr, a.k);
        const uint4* const xp = reinterpret_cast<const uint4*>(xr + row.head);
        const bool single = at < row.head || at >= EACH - row.tail;
        const int64_t single_at = at < row.head ? at : a.k - EACH + at;
        const float x1 = single ? to_f32(xr[single_at]) : 0.0f;
        uint32_t top = __float_as_uint(x1) & 0x7fffffffu;
        for (int p = at; p < row.pieces; p += EACH) top = max(top, q_largest<TX>(__ldg(xp + p)));
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) part[warp] = top;
        __syncthreads();
        top = part[t * (GV_WARPS / M)];
#pragma unroll
        for (int i = 1; i < GV_WARPS / M; ++i) top = max(top, part[t * (GV_WARPS / M) + i]);
        const q_row q(top);
        int8_t* const qr = xs + t * kp;
        const bool whole = row.head % N == 0;   // (kp is a multiple of 16)
        for (int p = at; p < row.pieces; p += EACH) q_store<TX>(qr + row.head + p * N, whole, __ldg(xp + p), q);
        if (single) qr[single_at] = (int8_t)q.integer(x1);
        if (at == 0) sx[t] = q.scale;
    }
    __syncthreads();
    for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
        int acc[M] = {};
        const int64_t row = row_of(g);
        const float ws = __ldg(a.w_scale + row), b = a.bias ? __ldg(a.bias + row) : 0.0f;
        for (int c0 = 0; c0 < chunks; c0 += GV_AHEAD) {
            if (c0 > 0) fetch(c0);
#pragma unroll
            for (int c = 0; c < GV_AHEAD; ++c)
                if (const int off = (c0 + c) * 512 + lane * 16; off < k16) gv_add<M>(acc, w[c], xs, kp, off);
        }
        if (lane < rest) {
            const int wb = wr[k16 + lane];
#pragma unroll
            for (int t = 0; t < M; ++t) acc[t] += wb * xs[t * kp + k16 + lane];
        }
        if (g + gridDim.x < groups) {
            wr = a.W + row_of(g + gridDim.x) * a.ldw;
            fetch(0);
        }
#pragma unroll
        for (int t = 0; t < M; ++t) {
            const int sum = __reduce_add_sync(0xffffffffu, acc[t]);
            if (lane == t && g * GV_WARPS + warp < a.n) {
                const float v = fmaf(__fmul_rn(sx[t], ws), (float)sum, b);
                static_cast<TY*>(a.y)[t * a.ldy + row] = from_f32<TY>(a.relu ? relu_ref(v) : v);
            }
        }
    }
}

template <typename TX, typename TY, int M> int gv_launch(s2v_ctx* ctx, cudaStream_t st, const GvArgs& a)
{
    const int64_t groups = (a.n + GV_WARPS - 1) / GV_WARPS, cap = (int64_t)ctx->sm_count * 4;
    S2V_CUDA_OK(ctx, s2v_allow_shared(gemv_i8_kernel<TX, TY, M>, GV_SMEM));
    gemv_i8_kernel<TX, TY, M><<<(unsigned)(groups < cap ? groups : cap), GV_THREADS, (size_t)M * a.kp, st>>>(a);
    S2V_CHECK_LAUNCH(ctx, "gemv_i8_kernel");
    return S2V_OK;
}
template <typename TX> int gv_by_size(s2v_ctx* ctx, cudaStream_t st, int y_type, const GvArgs& a)
{
    return s2v_by_dtype(y_type, [&](auto type) {
        using TY = decltype(type);
        return a.m == 1 ? gv_launch<TX, TY, 1>(ctx, st, a) : gv_launch<TX, TY, 2>(ctx, st, a);
    });
}

// ---------------------------------------------------------------- few tiles of outputs: k split among a cluster
// A CTA multiplies 128 weight rows (the rows of the accumulator) by NT tokens over its share of k; the integers of the shares are added through
// the cluster's shared memory, each CTA finishing an equal part of the tokens.  (Integer sums: the order does not matter.)
constexpr int GS_EPI = 8, GS_THREADS = 32 * (2 + GS_EPI);   // epilogue warps: two for each quarter of the weight rows, sharing the tokens
template <int NT> struct GsCfg {
    static constexpr uint32_t W_BYTES = 128 * 128, STAGE = W_BYTES + NT * 128;
    static constexpr int STAGES = NT <= 32 ? 5 : NT == 64 ? 4 : 3;   // about 100 KB: two CTAs an SM
    static constexpr uint32_t TM_COLS = NT < 32 ? 32 : NT;
    static constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);   // s32 <- s8 x s8, M = 128, N = NT
    static constexpr uint32_t OFF_SCALE = STAGES * STAGE;          // of the tokens
    static constexpr uint32_t OFF_BAR = OFF_SCALE + NT * 4;
    enum { FULL = 0, EMPTY = FULL + STAGES, DONE = EMPTY + STAGES, BARS = DONE + 1 };
    static constexpr uint32_t OFF_MISC = OFF_BAR + 8 * BARS;
    static constexpr uint32_t SMEM = OFF_MISC + 16 + 1024;
    static_assert(NT * 128 * 4 <= STAGES * STAGE, "the accumulator lies where the panels were");
};
struct GsArgs {
    int64_t m, n, ldc;
    int kblocks, last_steps, n_tiles, ctas;
    uint32_t bytes;   // of a panel: the weights', and the tokens' that there are (the products of the others are not looked at)
    const float* a_scale;
    const float* b_scale;
    const float* bias;
    void* C;
    int relu;
    s2v_device_status* status;
};

__device__ __forceinline__ void gs_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        :
        : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <typename T, int NT>
__global__ void __launch_bounds__(GS_THREADS) gemm_i8_split_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const GsArgs a)
{
    using Cfg = GsCfg<NT>;
    constexpr int STAGES = Cfg::STAGES;
    extern __shared__ unsigned char gs_raw[];
    unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(gs_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t smem0 = smem_u32(smem);
    const auto bar = [&](int i) { return smem0 + Cfg::OFF_BAR + 8u * (uint32_t)i; };
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::OFF_MISC);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_MISC + 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)(blockIdx.x % (unsigned)a.ctas), tile = (int)(blockIdx.x / (unsigned)a.ctas), tn = tile % a.n_tiles, tm = tile / a.n_tiles;
    const int k0 = (int)((int64_t)rank * a.kblocks / a.ctas), k1 = (int)((int64_t)(rank + 1) * a.kblocks / a.ctas), steps_k = k1 - k0;   // (at least one panel)
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) tc_mbar_init(bar(Cfg::FULL + i), 1), tc_mbar_init(bar(Cfg::EMPTY + i), 1);
        tc_mbar_init(bar(Cfg::DONE), 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&map_w);
        tma_prefetch_map(&map_x);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(Cfg::TM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    const int row = (warp & 3) * 32 + lane;                     // epilogue: this thread's weight row
    const int64_t col = (int64_t)tn * 128 + row;
    int* const mine = reinterpret_cast<int*>(smem);             // [NT][128]
    float* const token_scale = reinterpret_cast<float*>(smem + Cfg::OFF_SCALE);
    float sw = 0.0f, bias = 0.0f;
    bool done = true;
    const int half = (warp - 2) >> 2;
    const int tokens = (int)min((int64_t)NT, a.m - (int64_t)tm * NT);
    T* const out = static_cast<T*>(a.C) + (int64_t)tm * NT * a.ldc + col;
    const float least = a.relu ? 0.0f : -INFINITY;
    const auto put = [&](int t, int sum) {
        float v = fmaf(__fmul_rn(token_scale[t], sw), (float)sum, bias);
        v = v < least ? least : v;   // (NaN stays)
        if (t < tokens && col < a.n) out[t * a.ldc] = from_f32<T>(v);
    };

    if (warp == 0) {   // copies: the first weights before the tokens, which a kernel in front may still be writing
        const int ahead = min(STAGES, steps_k);
        if (tc_elect())
            for (int i = 0; i < ahead; ++i) {
                mbar_expect(bar(Cfg::FULL + i), a.bytes);
                tma_load_2d(smem0 + (uint32_t)i * Cfg::STAGE, &map_w, (k0 + i) * 128, tn * 128, bar(Cfg::FULL + i));
            }
        __syncwarp();
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if (tc_elect())
            for (int i = 0; i < ahead; ++i) tma_load_2d(smem0 + (uint32_t)i * Cfg::STAGE + Cfg::W_BYTES, &map_x, (k0 + i) * 128, tm * NT, bar(Cfg::FULL + i));
        __syncwarp();
        int it = ahead;
        for (; it < steps_k; ++it) {
            const int s = it % STAGES;
            if (!(done = tc_wait(bar(Cfg::EMPTY + s), (uint32_t)(it / STAGES - 1) & 1u, abort_flag, a.status, 74))) break;
            if (tc_elect()) {
                mbar_expect(bar(Cfg::FULL + s), a.bytes);
                tma_load_2d(smem0 + (uint32_t)s * Cfg::STAGE, &map_w, (k0 + it) * 128, tn * 128, bar(Cfg::FULL + s));
                tma_load_2d(smem0 + (uint32_t)s * Cfg::STAGE + Cfg::W_BYTES, &map_x, (k0 + it) * 128, tm * NT, bar(Cfg::FULL + s));
            }
            __syncwarp();
        }
        // no copy may arrive once the CTA has gone: where a wait gave up, the ones under way are waited for here (bounded like every wait)
        if (!done || *abort_flag)
            for (int i = max(0, it - STAGES); i < it; ++i) {
                int spins = 0;
                while (!tc_mbar_try(bar(Cfg::FULL + i % STAGES), (uint32_t)(i / STAGES) & 1u))
                    if (++spins > TC_WAIT_LIMIT) break;
            }
    } else if (warp == 1) {   // products
        int it = 0;
        for (; it < steps_k; ++it) {
            const int s = it % STAGES;
            if (!(done = tc_wait(bar(Cfg::FULL + s), (uint32_t)(it / STAGES) & 1u, abort_flag, a.status, 75))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (tc_elect()) {
                const uint64_t dw = tc_b_desc(smem0 + (uint32_t)s * Cfg::STAGE), dx = tc_b_desc(smem0 + (uint32_t)s * Cfg::STAGE + Cfg::W_BYTES);
                const int steps = k0 + it + 1 == a.kblocks ? a.last_steps : 4;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    if (ks < steps) gs_mma(tmem, dw + 2u * ks, dx + 2u * ks, Cfg::IDESC, it > 0 || ks > 0);
                asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar(Cfg::EMPTY + s)) : "memory");
                if (it + 1 == steps_k) asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar(Cfg::DONE)) : "memory");
            }
            __syncwarp();
        }
        if (!done || *abort_flag)   // products under way read shared memory and write tensor memory
            for (int i = max(0, it - STAGES); i < it; ++i) {
                int spins = 0;
                while (!tc_mbar_try(bar(Cfg::EMPTY + i % STAGES), (uint32_t)(i / STAGES) & 1u))
                    if (++spins > TC_WAIT_LIMIT) break;
            }
    } else {
        asm volatile("griddepcontrol.wait;" ::: "memory");   // the tokens' scales
        for (int t = (int)threadIdx.x - 64; t < NT; t += 32 * GS_EPI) token_scale[t] = (int64_t)tm * NT + t < a.m ? a.a_scale[(int64_t)tm * NT + t] : 0.0f;
        if (col < a.n) sw = __ldg(a.b_scale + col), bias = a.bias ? __ldg(a.bias + col) : 0.0f;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * GS_EPI) : "memory");
        done = tc_wait(bar(Cfg::DONE), 0, abort_flag, a.status, 76);
        if (done) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int h = 16 * half; h < NT; h += 32) {
                uint32_t v[16];
                tc_ld_cols16(tmem + (uint32_t)h + ((uint32_t)(warp & 3) << 21), v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (a.ctas == 1) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) put(h + j, (int)v[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) mine[(h + j) * 128 + row] = (int)v[j];   // (every panel has been read)
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    // every CTA of the cluster comes here, whatever its waits gave
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::TM_COLS) : "memory");
    if (warp >= 2 && done && a.ctas > 1) {
        uint32_t from[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
            if (c < a.ctas) asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from[c]) : "r"(smem_u32(mine + row)), "r"(c));
        const int share = NT / a.ctas / 2, t0 = rank * 2 * share + half * share, t1 = t0 + share;
        constexpr int G = NT < 32 ? 2 : NT < 128 ? 4 : 8;   // tokens whose sums are on their way at once (a load from another CTA takes as long as one from L2)
        for (int t = t0; t < t1; t += G) {
            int part[G][8];
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    part[g][c] = 0;
                    if (c < a.ctas && t + g < t1) asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(part[g][c]) : "r"(from[c] + (uint32_t)(t + g) * 512u) : "memory");
                }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                int sum = 0;
#pragma unroll
                for (int c = 0; c < 8; ++c) sum += part[g][c];
                if (t + g < t1) put(t + g, sum);
            }
        }
    }
    __syncwarp();
    // no CTA leaves while another reads its sums
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, int NT> int gs_launch(s2v_ctx* ctx, cudaStream_t st, const s2v_gemm_i8_args& g, int ctas, bool dependent)
{
    using Cfg = GsCfg<NT>;
    CUtensorMap map_w, map_x;
    const int64_t up = (g.k + 15) / 16 * 16;
    const int box = (int)(g.m < NT ? g.m : NT);   // (rows of zeros that the copy makes up take longer than none: 8 tokens 9.9 us)
    if (!s2v_byte_matrix_map(&map_w, g.B, g.n, g.k, g.n > 1 ? g.ldb : up, 128) || !s2v_byte_matrix_map(&map_x, g.A, g.m, g.k, g.m > 1 ? g.lda : up, box))
        return s2v_fail(ctx, S2V_ERR_CUDA, "gemm_i8: the driver did not take a matrix's tensor map");
    const int64_t nt = (g.n + 127) / 128, tiles = nt * ((g.m + NT - 1) / NT);
    if (tiles * ctas > INT32_MAX / 2) return s2v_fail(ctx, S2V_ERR_UNSUPPORTED, "gemm_i8: more than 2^30 tiles of outputs");
    GsArgs a;
    a.m = g.m, a.n = g.n, a.ldc = g.ldc;
    a.kblocks = (int)((g.k + 127) / 128);
    a.last_steps = (int)((g.k - 128 * (int64_t)(a.kblocks - 1) + 31) / 32);
    a.n_tiles = (int)nt, a.ctas = ctas, a.bytes = Cfg::W_BYTES + (uint32_t)box * 128;
    a.a_scale = g.a_scale, a.b_scale = g.b_scale, a.bias = g.bias, a.C = g.C, a.relu = g.relu;
    a.status = ctx->dstatus_dev;
    S2V_CUDA_OK(ctx, s2v_allow_shared(gemm_i8_split_kernel<T, NT>, Cfg::SMEM));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * ctas));
    cfg.blockDim = dim3(GS_THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 2 : 1;
    S2V_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, gemm_i8_split_kernel<T, NT>, map_w, map_x, a));
    S2V_CHECK_LAUNCH(ctx, "gemm_i8_split_kernel");
    return S2V_OK;
}

}  // namespace

bool s2v_gemv_i8_takes(int64_t m, int64_t n, int64_t k)
{
    return m <= 2 && k > 0 && n > 0 && m * ((k + 15) / 16 * 16) <= (int64_t)GV_SMEM;
}

int s2v_launch_gemv_i8(s2v_ctx* ctx, cudaStream_t st, int x_type, const s2v_gemm_i8_args& g)
{
    const GvArgs a{g.n, g.k, g.lda, g.n > 1 ? g.ldb : 0, g.ldc, (int)g.m, (int)((g.k + 15) / 16 * 16), g.A, g.a_scale, g.B, g.b_scale, g.bias, g.relu, g.C};
    if (x_type < 0) return gv_by_size<int8_t>(ctx, st, g.c_type, a);
    return s2v_by_dtype(x_type, [&](auto type) { return gv_by_size<decltype(type)>(ctx, st, g.c_type, a); });
}

// the split form for a call: tokens of a tile, tiles, and CTAs that share a tile's k
struct GsPlan {
    int nt, ctas;
    int64_t tiles, kblocks;
    GsPlan(const s2v_ctx* ctx, const s2v_gemm_i8_args& g)
    {
        nt = g.m <= 16 ? 16 : g.m <= 32 ? 32 : g.m <= 64 ? 64 : 128;
        tiles = (g.n + 127) / 128 * ((g.m + nt - 1) / nt);
        kblocks = (g.k + 127) / 128;
        // A CTA an SM, two where k is long (16 tokens, n = 4096: k = 4096 6.7 us with four CTAs a tile, 8.3 with eight; 4096 tokens of k = 14336 the same, 14336 x 14336 40.5 with
        // one CTA a tile, 36.5 with two)
        const int64_t most = ctx->sm_count * (kblocks >= 64 ? 2 : 1);
        ctas = 1;
        while (ctas < 8 && tiles * ctas * 2 <= most && kblocks >= 4 * ctas) ctas *= 2;
    }
};

float s2v_gemm_i8_split_cost(const s2v_ctx* ctx, const s2v_gemm_i8_args& g)
{
    const GsPlan p(ctx, g);
    const float each = (float)p.kblocks / p.ctas, waves = (float)((p.tiles * p.ctas + ctx->sm_count - 1) / ctx->sm_count);
    if (g.m > 64 && p.tiles > ctx->sm_count) return INFINITY;   // (nothing to gain: there are enough tiles)
    const float fixed = p.nt <= 32 ? 4.0f : p.nt == 64 ? 4.5f : 5.6f, panel = p.nt <= 32 ? .34f : p.nt == 64 ? .38f : .46f, outputs = (p.ctas > 1 ? .05f : .012f) * p.nt / p.ctas;
    return fixed + outputs + panel * each * (1.0f + .7f * (waves - 1.0f)) + outputs * (waves - 1.0f);
}

int s2v_launch_gemm_i8_split(s2v_ctx* ctx, cudaStream_t st, const s2v_gemm_i8_args& g, bool dependent)
{
    const GsPlan p(ctx, g);
    const int NT = p.nt, ctas = p.ctas;
    return s2v_by_dtype(g.c_type, [&](auto type) {
        using T = decltype(type);
        if (NT == 16) return gs_launch<T, 16>(ctx, st, g, ctas, dependent);
        if (NT == 32) return gs_launch<T, 32>(ctx, st, g, ctas, dependent);
        if (NT == 64) return gs_launch<T, 64>(ctx, st, g, ctas, dependent);
        return gs_launch<T, 128>(ctx, st, g, ctas, dependent);
    });
}
