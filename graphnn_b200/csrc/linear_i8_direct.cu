// dW = dy^T (scale q) for layers of few outputs over many rows, straight from dy and the 8-bit rows: what linear_i8_grad.cu writes to memory in 16 bits first, and
// reads again, goes to shared memory only.
//
// A CTA takes a share of the rows and a tile of dW of 256 x 128 or 128 x 256.  Sixteen warps load 32 rows at a time (a panel), multiply dy by the rows' scales, and put
// both into shared memory in 16 bits (fp32 as three bf16 numbers) as they lie, a row of 128 bytes for each 64 columns, 128-byte swizzle; the first one issues the
// products, which read both operands across k.  The numbers come by tensor-map copies, two panels or more ahead: a thread's own loads or 16-byte copies under way are waited for
// at the fence between its stores and the products (491,520 x 256 x 128 fp32: 294 and 326 us).  A sum stays in tensor memory for some 32 instructions only
// (mm16.cu says why); the warps add it up in registers, half of what the SM has, which is why no warp is set aside for the products.
#include <algorithm>
#include <cstring>

#include "f32x2.cuh"
#include "linear_i8_grad.cuh"
#include "tcgen05_pair.cuh"
#include "tma.cuh"

namespace
{

constexpr int LD_ROWS = 32, LD_WARPS = 16, LD_THREADS = 32 * LD_WARPS;   // rows of a panel
constexpr uint32_t LD_BLOCK = LD_ROWS * 128;                                   // bytes of a panel's 64 columns
constexpr int LD_STAGES = 4, LD_AHEAD = 4, LD_SCALES = 1024;   // operand panels and panels on their way, at most; rows' scales at a time
constexpr int LD_BARS = 2 * LD_STAGES + 4 + LD_AHEAD;
constexpr size_t LD_SHARED = 226 * 1024;

struct LdArgs {
    int64_t m, n, k, lddy, ldq, share;
    const void* dy;
    const int8_t* q;
    const float* scale;
    const float* factor;     // of columns of dy (fp16), or NULL
    int n_tiles, tile_n, tile_k;
    int a_blocks, b_blocks;  // of 64 columns: 2 or 4 of dy, 1, 2 or 4 of q
    int stages, ahead, chunk;   // operand panels; panels on their way; panels of an accumulator
    uint32_t idesc;
    float* part;             // [shares][n][pitch]
    int64_t pitch;
    float* columns;          // [shares][n]: sums of dy, or NULL
    s2v_device_status* status;
};

// ANB: blocks of dy in a panel (2 or 4); a thread has eight columns of one or two of a panel's rows.
template <typename T, int ANB>
__global__ void __launch_bounds__(LD_THREADS, 1) linear_i8_direct_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_q, const LdArgs a)
{
    constexpr int PARTS = sizeof(T) == 4 ? 3 : 1, GROUPS = ANB * 8, LANES = LD_WARPS * 32 / GROUPS, HALVES = ANB / 2, U = LD_ROWS / LANES;   // HALVES: 128 rows of dW each; U: rows of a thread
    constexpr int BU = 2 / HALVES;   // rows of q of a thread, at most
    using H = typename std::conditional<std::is_same<T, __half>::value, __half, __nv_bfloat16>::type;
    extern __shared__ unsigned char ld_raw[];
    unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ld_raw) + 1023) & ~(uintptr_t)1023);
    constexpr int RAW = (int)sizeof(T) * 8 / 16;                    // 16-byte pieces of eight columns
    constexpr uint32_t WAY_DY = LD_ROWS * ANB * 64 * sizeof(T);   // bytes of a panel on its way; then q's
    const uint32_t smem0 = smem_u32(smem), stage_bytes = (uint32_t)(PARTS * ANB + a.b_blocks) * LD_BLOCK, way_bytes = WAY_DY + (uint32_t)(LD_ROWS * a.b_blocks * 64),
                   off_way = (uint32_t)a.stages * stage_bytes, off_scale = off_way + (uint32_t)a.ahead * way_bytes, off_bar = off_scale + 2 * LD_SCALES * 4;
    float* const scales = reinterpret_cast<float*>(smem + off_scale);   // of two spans of LD_SCALES rows
    const auto full = [&](int s) { return smem0 + off_bar + 8u * (uint32_t)s; };
    const auto empty = [&](int s) { return smem0 + off_bar + 8u * (uint32_t)(LD_STAGES + s); };
    const auto done = [&](int s) { return smem0 + off_bar + 8u * (uint32_t)(2 * LD_STAGES + s); };
    const auto read = [&](int s) { return smem0 + off_bar + 8u * (uint32_t)(2 * LD_STAGES + 2 + s); };
    const auto here = [&](int s) { return smem0 + off_bar + 8u * (uint32_t)(2 * LD_STAGES + 4 + s); };
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + off_bar + 8 * LD_BARS);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + off_bar + 8 * LD_BARS + 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) tc_mbar_init(full(i), LD_WARPS), tc_mbar_init(empty(i), 1);
        for (int i = 0; i < 2; ++i) tc_mbar_init(done(i), 1), tc_mbar_init(read(i), LD_WARPS);
        for (int i = 0; i < a.ahead; ++i) tc_mbar_init(here(i), 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    const int share = (int)blockIdx.x, tile = (int)blockIdx.y;
    const int64_t n0 = (int64_t)(tile % a.n_tiles) * a.tile_n, k0 = (int64_t)(tile / a.n_tiles) * a.tile_k;
    const int64_t from = share * a.share, to = min(a.m, from + a.share);
    const int panels = (int)((to - from + LD_ROWS - 1) / LD_ROWS), chunks = (panels + a.chunk - 1) / a.chunk, cols = a.b_blocks * 64;   // columns of an accumulator

    bool ok = true;
    // Panel p on its way, by one thread; where rows or columns end, zeros (shares end at multiples of a panel).
    const auto ask = [&](int p, int slot) {
        if (p >= panels) return;
        mbar_expect(here(slot), way_bytes);
        const uint32_t to_smem = smem0 + off_way + (uint32_t)slot * way_bytes;
        tma_load_2d(to_smem, &map_dy, (int)n0, (int)from + p * LD_ROWS, here(slot));
        tma_load_2d(to_smem + WAY_DY, &map_q, (int)k0, (int)from + p * LD_ROWS, here(slot));
    };
    // The products of panel p, by warp 0, which then asks for the panel that takes its place on the way: every warp has read it.
    int at_stage = 0, at_in = 0, at_chunk = 0;
    uint32_t at_phase = 0;
    const auto multiply = [&](int p, int slot) {
        const int buf = at_chunk & 1;
        if (at_in == 0 && at_chunk >= 2 && !(ok = ok && tc_wait(read(buf), (uint32_t)(at_chunk / 2 - 1) & 1u, abort_flag, a.status, 96))) return;
        if (!(ok = ok && tc_wait(full(at_stage), at_phase, abort_flag, a.status, 97))) return;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const bool last = at_in + 1 == a.chunk || p + 1 == panels;
        if (tc_elect()) {
            const uint32_t at = smem0 + (uint32_t)at_stage * stage_bytes;
            const uint64_t db = tc_desc_across<LD_BLOCK>(at + (uint32_t)(PARTS * ANB) * LD_BLOCK);
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    const uint64_t da = tc_desc_across<LD_BLOCK>(at + (uint32_t)(q * ANB + 2 * h) * LD_BLOCK);
#pragma unroll
                    for (int ks = 0; ks < LD_ROWS / 16; ++ks)   // 16 rows of 128 bytes
                        tc_mma_f16<false>(tmem + (uint32_t)(buf * 256 + h * cols), da + 128u * ks, db + 128u * ks, a.idesc, at_in > 0 || q > 0 || ks > 0);
                }
            tc_commit<false>(empty(at_stage));
            if (last) tc_commit<false>(done(buf));
            ask(p + a.ahead, slot);
        }
        __syncwarp();
        if (++at_stage == a.stages) at_stage = 0, at_phase ^= 1;
        if (last) at_in = 0, ++at_chunk;
        else ++at_in;
    };
    int multiplied = 0;   // panels, of warp 0
    {
        const int group = threadIdx.x % GROUPS, first_row = threadIdx.x / GROUPS;
        const int64_t col = n0 + group * 8;
        const int have = (int)max((int64_t)0, min((int64_t)8, min(a.n, n0 + a.tile_n) - col));   // of the thread's columns
        const int b_groups = a.b_blocks * 8, b_lanes = LD_WARPS * 32 / b_groups, b_group = threadIdx.x % b_groups, b_first = threadIdx.x / b_groups;
        float factor[8];
        uint64_t sums[4] = {};   // (zeros)
#pragma unroll
        for (int e = 0; e < 8; ++e) factor[e] = a.factor && e < have ? a.factor[col + e] : 1.0f;
        // scales of a span of rows, a turn of it ahead
        const auto span = [&](int i) {
            for (int r = (int)threadIdx.x; r < LD_SCALES; r += LD_THREADS) {
                const int64_t at = from + (int64_t)i * LD_SCALES + r;
                scales[(i & 1) * LD_SCALES + r] = at < to ? a.scale[at] : 0.0f;
            }
        };
        const auto place = [&](uint32_t block0, int g, int row) { return block0 + (uint32_t)(g >> 3) * LD_BLOCK + (uint32_t)(row * 128 + 16 * ((g & 7) ^ (row & 7))); };
        const auto store16 = [&](uint32_t at, const uint32_t* h) {
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
        };
        // Sums of a finished chunk, onto those before: a quarter of the lanes and a fourth of the columns a warp.
        const int quarter = warp & 3, fourth = warp >> 2, all = HALVES * cols, mine = all / 4;   // columns of a warp: 16, 32 or 64
        float y[64];
#pragma unroll
        for (int j = 0; j < 64; ++j) y[j] = 0.0f;
        const auto take = [&](int c) {
            if (!(ok = ok && tc_wait(done(c & 1), (uint32_t)(c / 2) & 1u, abort_flag, a.status, 98))) return;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at = tmem + (uint32_t)((c & 1) * 256 + fourth * mine) + ((uint32_t)quarter << 21);
#pragma unroll
            for (int j = 0; j < 64; j += 16) {
                if (j >= mine) break;
                uint32_t v[16];
                tc_ld_cols16(at + (uint32_t)j, v);
                tc_wait_loads(v);
#pragma unroll
                for (int e = 0; e < 16; ++e) y[j + e] += __uint_as_float(v[e]);
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) tc_mbar_arrive(read(c & 1));
        };
        int s = 0, taken = 0, in = 0, c = 0, slot = 0;
        uint32_t phase = 0, way_phase = 0;
        span(0);
        if (threadIdx.x == 0)
            for (int p = 0; p < a.ahead; ++p) ask(p, p);
        __syncthreads();   // (scales)
        for (int p = 0; p < panels; ++p) {
            // the next span's scales take the place of the last one's, which every warp has done with: half a span ago at least it arrived behind them, and
            // half a span goes by before they are used
            if ((p & (LD_SCALES / LD_ROWS - 1)) == LD_SCALES / LD_ROWS / 2) span(p / (LD_SCALES / LD_ROWS) + 1);
            if (p >= a.stages && !(ok = tc_wait(empty(s), phase ^ 1u, abort_flag, a.status, 99))) break;
            const uint32_t at = smem0 + (uint32_t)s * stage_bytes;
            if (!(ok = tc_wait(here(slot), way_phase, abort_flag, a.status, 95))) break;
            const unsigned char* const way = smem + off_way + (uint32_t)slot * way_bytes;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int row = first_row + u * LANES;
                const float by = scales[(p * LD_ROWS + row) & (2 * LD_SCALES - 1)];
                uint64_t f[4];
#pragma unroll
                for (int j = 0; j < RAW; ++j) f2_unpack<T>(*reinterpret_cast<const uint4*>(way + (uint32_t)(row * ANB * 64 + group * 8) * (uint32_t)sizeof(T) + 16 * j), f + j * PIECE<T> / 2);
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) sums[e] = f2_add(sums[e], f[e]), f[e] = f2_mul(f[e], f2_of(by, by));
                if (a.factor) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[e] = f2_mul(f[e], f2_of(factor[2 * e], factor[2 * e + 1]));
                }
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 v = f2_get(f[j]);
                        // (of three parts the first is cut, which no number is too large for; with 8-bit integers as the other operand no product of parts is left out)
                        h[j] = PARTS > 1 && q == 0 ? __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x7632) : pack_16bit<H>(v.x, v.y);
                        if (q + 1 < PARTS) f[j] = f2_add(f[j], f2_of(-__uint_as_float(h[j] << 16), -__uint_as_float(h[j] & 0xffff0000u)));
                    }
                    store16(place(at + (uint32_t)(q * ANB) * LD_BLOCK, group, first_row + u * LANES), h);
                }
            }
#pragma unroll
            for (int u = 0; u < BU; ++u) {
                const int row = b_first + u * b_lanes;
                if (row >= LD_ROWS) continue;
                const uint2 bytes = *reinterpret_cast<const uint2*>(way + WAY_DY + (uint32_t)(row * a.b_blocks * 64 + b_group * 8));
                uint64_t f[4];
                uint32_t h[4];
                f2_unpack8(bytes.x, f), f2_unpack8(bytes.y, f + 2);
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = pack_16bit<H>(f2_get(f[j]).x, f2_get(f[j]).y);
                store16(place(at + (uint32_t)(PARTS * ANB) * LD_BLOCK, b_group, row), h);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tc_mbar_arrive(full(s));
            if (++s == a.stages) s = 0, phase ^= 1;
            if (warp == 0) multiply(p, slot), ++multiplied;
            if (!ok) break;
            if (++slot == a.ahead) slot = 0, way_phase ^= 1;
            // a chunk is taken while the next one's panels are being multiplied
            if (++in == a.chunk) in = 0, ++c;
            if (c > taken && in + 1 == a.chunk) take(taken++);
            if (!ok) break;
        }
        for (; ok && taken < chunks; ++taken) take(taken);
        // products under way read shared memory and write tensor memory, copies write shared memory: where a wait gave up, the last ones of every place
        if (warp == 0 && (!ok || *abort_flag))
            for (int i = max(0, multiplied); i < min(panels, multiplied + a.ahead); ++i) {
                int spins = 0;
                while (!tc_mbar_try(here(i % a.ahead), (uint32_t)(i / a.ahead) & 1u))
                    if (++spins > TC_WAIT_LIMIT) break;
            }
        if (warp == 0 && (!ok || *abort_flag))
            for (int i = max(0, multiplied - a.stages); i < multiplied; ++i) {
                int spins = 0;
                while (!tc_mbar_try(empty(i % a.stages), (uint32_t)(i / a.stages) & 1u))
                    if (++spins > TC_WAIT_LIMIT) break;
            }
        if (ok) {
            const int row = quarter * 32 + lane;
#pragma unroll
            for (int j = 0; j < 64; j += 4) {
                if (j >= mine) break;
                const int at = fourth * mine + j, h = at / cols;   // of all columns; which 128 rows of the tile
                const int64_t i = n0 + h * 128 + row, l = k0 + at % cols;
                if (i < min(a.n, n0 + a.tile_n) && l < a.k) *reinterpret_cast<float4*>(a.part + ((int64_t)share * a.n + i) * a.pitch + l) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
            }
        }
        // sums of dy: threads with the same columns, through the first stage's place once its products are done (all of them are: every chunk was taken)
        __syncthreads();
        float* const of = reinterpret_cast<float*>(smem);
        if (a.columns && k0 == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<uint64_t*>(of + first_row * (GROUPS * 8) + group * 8 + 2 * e) = sums[e];
        }
        __syncthreads();
        if (a.columns && k0 == 0 && ok)
            for (int j = threadIdx.x; j < GROUPS * 8; j += LD_WARPS * 32)
                if (n0 + j < min(a.n, n0 + a.tile_n)) {
                    float t = 0.0f;
                    for (int r = 0; r < LANES; ++r) t += of[r * (GROUPS * 8) + j];
                    a.columns[(int64_t)share * a.n + n0 + j] = t;
                }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// dW = alpha * the shares' sums, added in a fixed order: four columns a thread, a quarter of the shares each
template <typename T> __global__ void __launch_bounds__(256) linear_i8_shares_kernel(int shares, int64_t n, int64_t k, int64_t pitch, const float* __restrict__ part, const float* __restrict__ alpha,
                                                                                     T* __restrict__ dW, int64_t lddw)
{
    __shared__ float4 of[4][64];
    const int64_t per_row = pitch / 4, at = (int64_t)blockIdx.x * 64 + threadIdx.x % 64;
    const int g = threadIdx.x / 64;
    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (at < n * per_row) {
#pragma unroll 8
        for (int s = g; s < shares; s += 4) {
            const float4 f = __ldcs(reinterpret_cast<const float4*>(part) + s * n * per_row + at);
            t.x += f.x, t.y += f.y, t.z += f.z, t.w += f.w;
        }
    }
    of[g][threadIdx.x % 64] = t;
    __syncthreads();
    if (g || at >= n * per_row) return;
    const int64_t row = at / per_row, col = (at - row * per_row) * 4;
    float y[4] = {};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const float4 f = of[s][threadIdx.x];
        y[0] += f.x, y[1] += f.y, y[2] += f.z, y[3] += f.w;
    }
    const float by = alpha ? alpha[row] : 1.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e < k) dW[row * lddw + col + e] = from_f32<T>(by * y[e]);
}

// Tiles of dW: 256 x 128, or 128 x 256 where n is no more than 128.
struct LdShape {
    int64_t tile_n, tile_k, n_tiles, k_tiles, shares, share;
    LdShape(int64_t m, int64_t n, int64_t k, int64_t sms)
    {
        tile_n = n > 128 ? 256 : 128, tile_k = n > 128 ? 128 : 256;
        n_tiles = (n + tile_n - 1) / tile_n, k_tiles = (k + tile_k - 1) / tile_k;
        shares = std::max<int64_t>(1, std::min(sms / (n_tiles * k_tiles), m / (4 * LD_ROWS)));
        share = ((m + shares - 1) / shares + LD_ROWS - 1) / LD_ROWS * LD_ROWS;
        shares = (m + share - 1) / share;
    }
};

}  // namespace

bool linear_i8_direct_lies(int64_t m, int dy_type, const void* dy, int64_t lddy, const int8_t* q, int64_t ldq)
{
    return s2v_aligned16(dy) && s2v_aligned16(q) && (m <= 1 || (lddy * (int64_t)s2v_dtype_bytes(dy_type) % 16 == 0 && ldq % 16 == 0));
}
bool linear_i8_direct_takes(int64_t m, int64_t n, int64_t k, int dy_type)
{
    const int64_t tiles = n > 128 ? ((n + 255) / 256) * ((k + 127) / 128) : (k + 255) / 256;
    return tiles <= (dy_type == S2V_F32 ? 4 : 2) && m >= 4096;
}
size_t linear_i8_direct_floats(int64_t m, int64_t n, int64_t k) { return (size_t)LdShape(m, n, k, 148).shares * n * ((k + 7) / 8 * 8); }

int linear_i8_direct(s2v_ctx* ctx, cudaStream_t st, const linear_i8_grad_args& g, float* part, float* columns, int* shares)
{
    const LdShape shape(g.m, g.n, g.k, std::min(ctx->sm_count, 148));
    LdArgs a = {};
    a.m = g.m, a.n = g.n, a.k = g.k, a.lddy = g.lddy, a.ldq = g.ldq, a.share = shape.share;
    a.dy = g.dy, a.q = g.q, a.scale = g.scale, a.factor = g.factor;
    const int64_t es = (int64_t)s2v_dtype_bytes(g.dy_type);
    a.n_tiles = (int)shape.n_tiles, a.tile_n = (int)shape.tile_n, a.tile_k = (int)shape.tile_k;
    a.a_blocks = g.n > 128 ? 4 : 2;
    const int64_t widest = std::min(g.k, shape.tile_k);
    a.b_blocks = widest <= 64 ? 1 : widest <= 128 ? 2 : 4;
    const int parts = g.dy_type == S2V_F32 ? 3 : 1;
    const size_t stage = (size_t)(parts * a.a_blocks + a.b_blocks) * LD_BLOCK, fixed = 1024 + 2 * LD_SCALES * 4 + 8 * LD_BARS + 16;
    const size_t way = (size_t)LD_ROWS * (shape.tile_n * es + a.b_blocks * 64), left = LD_SHARED - fixed;
    a.ahead = (int)std::min<size_t>(LD_AHEAD, std::max<size_t>(2, (left - 2 * stage) / way));   // (in the largest form, of fp32, two of either fit)
    a.stages = (int)std::min<size_t>(LD_STAGES, (left - a.ahead * way) / stage);
    a.chunk = std::max(2, 16 / parts);   // 32 instructions, about
    const uint32_t type = g.dy_type == S2V_F16 ? 0u : 1u;
    a.idesc = (1u << 4) | (type << 7) | (type << 10) | (1u << 15) | (1u << 16) | ((uint32_t)(a.b_blocks * 64 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    a.part = part, a.pitch = (g.k + 7) / 8 * 8, a.columns = columns, a.status = ctx->dstatus_dev;
    *shares = (int)shape.shares;
    CUtensorMap map_dy, map_q;
    if (!s2v_matrix_map(&map_dy, (int)es, g.dy, g.m, g.n, g.lddy, a.tile_n, LD_ROWS) || !s2v_matrix_map(&map_q, 1, g.q, g.m, g.k, g.ldq, a.b_blocks * 64, LD_ROWS))
        return s2v_fail(ctx, S2V_ERR_CUDA, "linear_i8_grad: the driver did not take a matrix's tensor map");
    const dim3 grid((unsigned)shape.shares, (unsigned)(shape.n_tiles * shape.k_tiles));
    const auto go = [&](auto kernel) {
        S2V_CUDA_OK(ctx, s2v_allow_shared(kernel, LD_SHARED));
        kernel<<<grid, LD_THREADS, fixed + a.ahead * way + a.stages * stage, st>>>(map_dy, map_q, a);
        S2V_CHECK_LAUNCH(ctx, "linear_i8_direct_kernel");
        return (int)S2V_OK;
    };
    const int rc = s2v_by_dtype(g.dy_type, [&](auto type) {
        using T = decltype(type);
        return a.a_blocks == 4 ? go(linear_i8_direct_kernel<T, 4>) : go(linear_i8_direct_kernel<T, 2>);
    });
    if (rc != S2V_OK) return rc;
    return s2v_by_dtype(g.dy_type, [&](auto type) {
        using T = decltype(type);
        linear_i8_shares_kernel<T><<<(unsigned)((g.n * (a.pitch / 4) + 63) / 64), 256, 0, st>>>(*shares, g.n, g.k, a.pitch, part, g.alpha, static_cast<T*>(g.dW), g.lddw);
        S2V_CHECK_LAUNCH(ctx, "linear_i8_shares_kernel");
        return (int)S2V_OK;
    });
}
