// C = act((a_scale x b_scale) * (A B^T) + bias) for 8-bit A [m x k] and B [n x k]: tcgen05 matrix instructions with 32-bit integer accumulators.
//
// A persistent CTA per SM walks over tiles of 128 x BN outputs, or a pair of CTAs over tiles of 256 x 256: each keeps 128 rows of A and 128 of B,
// and one instruction multiplies all of A by all of B into both tensor memories.  (A CTA by itself needs 384 rows a tile: 94 bytes a cycle and SM from
// L2, more than it gives, and the tensor cores were busy 71 % of the time.)  One warp copies panels of 128 bytes along k (tensor maps, 128-byte swizzle; zeros
// outside the matrices) into a ring, one issues the products, eight take finished accumulators out of tensor memory, of which there are two, so
// that a tile's outputs are written under the next tile's products.
#include <cmath>
#include <cstring>

#include "gemm_i8.cuh"
#include "tcgen05_pair.cuh"
#include "tma.cuh"

namespace
{

constexpr int GI_EPI = 8;                              // epilogue warps
constexpr int GI_THREADS = 32 * (2 + GI_EPI);
constexpr int GI_PIECE = 64, GI_BOX = 32 * GI_PIECE;    // bytes of a row that an epilogue warp hands over at a time; of its 32 rows

template <int BN, bool PAIR> struct GiCfg {
    static constexpr int B_ROWS = PAIR ? BN / 2 : BN;   // of B, in this CTA's shared memory
    static constexpr uint32_t A_BYTES = 128 * 128, B_BYTES = B_ROWS * 128, STAGE = A_BYTES + B_BYTES;
    // (128 x 256 with four stages and one box: 491,520 x 256 outputs of bf16 over k = 128 85 us, with three and two 65; 300 x 11000 x 4096 18.9 and 19.7)
    static constexpr int STAGES = PAIR ? (BN == 256 ? 5 : 7) : BN == 256 ? 3 : BN == 128 ? 5 : 7, BOXES = 2;   // boxes of an epilogue warp
    static constexpr int ACCS = 2;   // accumulators (four of 128 columns: no faster)
    static constexpr uint32_t TM_COLS = ACCS * BN;
    static constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)((PAIR ? 256 : 128) >> 4) << 24);   // s32 <- s8 x s8, M = 128 or 256, N = BN
    static constexpr uint32_t OFF_OUT = STAGES * STAGE;                       // per epilogue warp: its boxes
    static constexpr uint32_t OFF_SCALE = OFF_OUT + GI_EPI * BOXES * GI_BOX;   // per epilogue warp: the scales of half a tile's channels, then their biases
    static constexpr uint32_t OFF_BAR = OFF_SCALE + GI_EPI * BN * 4;
    enum { FULL = 0, EMPTY = FULL + STAGES, DONE = EMPTY + STAGES, READ = DONE + ACCS, BARS = READ + ACCS };
    static constexpr uint32_t OFF_MISC = OFF_BAR + 8 * BARS;
    static constexpr uint32_t SMEM = OFF_MISC + 16 + 1024;                    // + slack to align the base to 1024 bytes
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct GiArgs {
    int64_t m, n, ldc;
    int kblocks, last_steps;        // panels along k; matrix instructions of the last one (32 bytes each)
    int m_tiles, n_tiles;
    const float* a_scale;
    const float* b_scale;
    const float* bias;
    void* C;
    int relu, boxes;                // boxes: the output has a tensor map (16-byte aligned rows)
    uint32_t bytes;                 // of a panel of this CTA
    s2v_device_status* status;
};

template <bool PAIR> __device__ __forceinline__ void gi_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
            :
            : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
            :
            : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
}
// fma(sa * s, v, b) of two accumulators, in packed fp32 arithmetic
__device__ __forceinline__ void gi_two(uint64_t sa, uint64_t s, uint64_t b, uint32_t v0, uint32_t v1, float& y0, float& y1)
{
    asm("{\n\t.reg .b64 v, s;\n\t"
        "mov.b64 v, {%5, %6};\n\t"
        "mul.rn.f32x2 s, %2, %3;\n\t"
        "fma.rn.f32x2 v, s, v, %4;\n\t"
        "mov.b64 {%0, %1}, v;\n\t}"
        : "=f"(y0), "=f"(y1)
        : "l"(sa), "l"(s), "l"(b), "f"((float)(int)v0), "f"((float)(int)v1));
}
// The accumulators of 32 rows by 64 bytes of outputs, COLS columns, as matrices of 8 rows by 16 bytes of outputs: lane l has word l % 4 of
// row l / 4 of each, which is as stmatrix wants it.
template <typename T> __device__ __forceinline__ void gi_fetch(uint32_t at, uint32_t* v)
{
#pragma unroll
    for (int h = 0; h < 2; ++h, at += 16u << 16) {
        if constexpr (sizeof(T) == 4)
            asm volatile("tcgen05.ld.sync.aligned.16x128b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                         : "=r"(v[8 * h]), "=r"(v[8 * h + 1]), "=r"(v[8 * h + 2]), "=r"(v[8 * h + 3]), "=r"(v[8 * h + 4]), "=r"(v[8 * h + 5]), "=r"(v[8 * h + 6]), "=r"(v[8 * h + 7])
                         : "r"(at)
                         : "memory");
        else
            asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                         : "=r"(v[16 * h]), "=r"(v[16 * h + 1]), "=r"(v[16 * h + 2]), "=r"(v[16 * h + 3]), "=r"(v[16 * h + 4]), "=r"(v[16 * h + 5]), "=r"(v[16 * h + 6]), "=r"(v[16 * h + 7]),
                           "=r"(v[16 * h + 8]), "=r"(v[16 * h + 9]), "=r"(v[16 * h + 10]), "=r"(v[16 * h + 11]), "=r"(v[16 * h + 12]), "=r"(v[16 * h + 13]), "=r"(v[16 * h + 14]), "=r"(v[16 * h + 15])
                         : "r"(at)
                         : "memory");
    }
}
// Where a column of half a tile stands in the table of scales: a lane's columns of one piece side by side.
template <typename T> __device__ __forceinline__ int gi_place(int c)
{
    if constexpr (sizeof(T) == 4) return (c & ~15) + 4 * (c & 3) + (c >> 2 & 3);
    else return (c & ~31) + 8 * (c >> 1 & 3) + 2 * (c >> 3 & 3) + (c & 1);
}
// The outputs, as 64-byte rows of a box whose 16-byte pieces are exchanged by the 64-byte swizzle, which keeps the stores free of bank conflicts.
// (With a row a lane every lane reads every scale and bias, 16 bytes for four columns of one row, and shared memory is what such an epilogue waits for:
// 491,520 x 256 outputs over k = 128 105 us in fp32 and 80 us in bf16; so 103 and 65.)
template <typename T, int HALF, bool RELU> __device__ __forceinline__ void gi_fill(unsigned char* box, const float* chan, const uint64_t* sa, const uint32_t* v)
{
    constexpr int PAIRS = 8 / sizeof(T), VALUES = 2 * PAIRS;   // of a lane's columns
    const int lane = threadIdx.x & 31;
    ulonglong2 s[PAIRS / 2], b[PAIRS / 2];
#pragma unroll
    for (int j = 0; j < PAIRS / 2; ++j)
        s[j] = reinterpret_cast<const ulonglong2*>(chan + VALUES * (lane & 3))[j], b[j] = reinterpret_cast<const ulonglong2*>(chan + HALF + VALUES * (lane & 3))[j];
    const uint32_t to = smem_u32(box) + (lane & 7) * GI_PIECE + 16 * ((lane >> 3) ^ (lane >> 1 & 3));
#pragma unroll
    for (int r = 0; r < 4; ++r) {   // 8 rows
        float y[VALUES];
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            const uint32_t* const from = v + r / 2 * (PAIRS * 4) + (sizeof(T) == 4 ? 4 * j + r % 2 : 4 * j + 2 * (r % 2));
            gi_two(sa[r], j & 1 ? s[j / 2].y : s[j / 2].x, j & 1 ? b[j / 2].y : b[j / 2].x, from[0], from[sizeof(T) == 4 ? 2 : 1], y[2 * j], y[2 * j + 1]);
        }
        if constexpr (RELU) {
#pragma unroll
            for (int u = 0; u < VALUES; ++u) y[u] = relu_ref(y[u]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(y[j]);
            else w[j] = pack_16bit<T>(y[2 * j], y[2 * j + 1]);
        }
        asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(to + r * 8 * GI_PIECE), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
}

// The outputs of 32 rows by COLS columns: into a box in shared memory, and from there by one copy that leaves out rows and 16-byte pieces which the
// matrix does not have.  (Written by the warp's own loads and stores, a product with few sums an output was bound by that: 491,520 x 256 outputs of fp32
// over k = 128 158 us.)
template <typename T, int HALF>
__device__ __forceinline__ void gi_write(const GiArgs& a, const CUtensorMap* map, unsigned char* box, const float* chan, int64_t row0, int64_t col0, const uint64_t* sa, const uint32_t* v)
{
    constexpr int COLS = GI_PIECE / sizeof(T), PER = 16 / sizeof(T);
    const int lane = threadIdx.x & 31;
    if (a.relu) gi_fill<T, HALF, true>(box, chan, sa, v);
    else gi_fill<T, HALF, false>(box, chan, sa, v);
    // (a copy that meets the end of a row inside 16 bytes writes zeros behind it, into what may be somebody else's)
    if (a.boxes && (col0 + COLS <= a.n || a.n % PER == 0)) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) tma_store_2d(map, (int)col0, (int)row0, smem_u32(box));
    } else {
        // Rows that start anywhere: 16 lanes a row, a word of four bytes each.  In a row of 16-bit numbers at an odd place a lane writes the second half of
        // its word with the first half of its neighbour's, the first lane the first number and the last lane the last one.
        __syncwarp();
        const int l = lane & 15, hi = lane >> 4;
        T* const to = static_cast<T*>(a.C) + (row0 + hi) * a.ldc + col0;
        const int cols = (int)min((int64_t)COLS, a.n - col0), rows = (int)min((int64_t)32, a.m - row0);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const unsigned char* const from = box + hi * GI_PIECE + u * 2 * GI_PIECE + 16 * ((l >> 2) ^ u) + 4 * (l & 3);   // (rows of this u have the same swizzle)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = hi + 2 * u + 8 * i;
                T* const at = to + (2 * u + 8 * i) * a.ldc;
                const uint32_t w = *reinterpret_cast<const uint32_t*>(from + i * 8 * GI_PIECE);
                if constexpr (sizeof(T) == 4) {
                    if (r < rows && l < cols) *reinterpret_cast<uint32_t*>(at + l) = w;
                } else {
                    uint16_t* const h = reinterpret_cast<uint16_t*>(at) + 2 * l;
                    const uint32_t next = __shfl_down_sync(0xffffffffu, w, 1);
                    if (r >= rows) continue;
                    if ((reinterpret_cast<uintptr_t>(h) & 2) == 0) {
                        if (2 * l + 1 < cols) *reinterpret_cast<uint32_t*>(h) = w;
                        else if (2 * l < cols) h[0] = (uint16_t)w;
                    } else {
                        if (l < 15 && 2 * l + 2 < cols) *reinterpret_cast<uint32_t*>(h + 1) = __byte_perm(w, next, 0x5432);
                        else if (2 * l + 1 < cols) h[1] = (uint16_t)(w >> 16);
                        if (l == 0) h[0] = (uint16_t)w;
                    }
                }
            }
        }
        // among copies a piece is a bulk group in any case: the wait before a box is filled counts groups, and this one's turn is over like a copy's
        // (without copies there is nothing to wait for: 20000 x 1021 of fp32 over k = 128, rows at odd places, 37.1 us with the groups, 36.7 without)
        if (a.boxes && lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        __syncwarp();
    }
}

template <typename T, int BN, bool PAIR>
__global__ void __launch_bounds__(GI_THREADS, 1) gemm_i8_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_c, const GiArgs a)
{
    using Cfg = GiCfg<BN, PAIR>;
    constexpr int STAGES = Cfg::STAGES, ACCS = Cfg::ACCS, CTAS = PAIR ? 2 : 1;
    extern __shared__ unsigned char gi_raw[];
    unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(gi_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t smem0 = smem_u32(smem);
    const auto bar = [&](int i) { return smem0 + Cfg::OFF_BAR + 8u * (uint32_t)i; };
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::OFF_MISC);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_MISC + 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = a.m_tiles * a.n_tiles, rank = PAIR ? (int)(blockIdx.x & 1) : 0, unit = (int)blockIdx.x / CTAS, units = (int)gridDim.x / CTAS;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) tc_mbar_init(bar(Cfg::FULL + i), 1), tc_mbar_init(bar(Cfg::EMPTY + i), 1);
        for (int i = 0; i < ACCS; ++i) tc_mbar_init(bar(Cfg::DONE + i), 1), tc_mbar_init(bar(Cfg::READ + i), GI_EPI * CTAS);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (a.kblocks > 0) tma_prefetch_map(&map_a), tma_prefetch_map(&map_b);
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(Cfg::TM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(Cfg::TM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (PAIR) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // both CTAs' barriers are there
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

    asm volatile("griddepcontrol.wait;" ::: "memory");   // A and its scales may come from a kernel in front
    if (warp == 0) {   // copies
        int it = 0;
        bool ok = true;
        for (int tile = unit; ok && tile < tiles; tile += units) {
            int tm, tn;
            tc_tile(tile, a.m_tiles, a.n_tiles, tm, tn);
            for (int kb = 0; kb < a.kblocks; ++kb, ++it) {
                const int s = it % STAGES;
                if (it >= STAGES && !(ok = tc_wait(bar(Cfg::EMPTY + s), (uint32_t)(it / STAGES - 1) & 1u, abort_flag, a.status, 70))) break;
                if (tc_elect()) {
                    const uint32_t at = smem0 + (uint32_t)s * Cfg::STAGE;
                    if constexpr (PAIR) {   // both CTAs' copies count on the first one's barrier, where the products are issued
                        if (rank == 0) mbar_expect(bar(Cfg::FULL + s), 2 * a.bytes);
                        const uint32_t b = tc_pair_first(bar(Cfg::FULL + s));
                        tma_load_2d_pair(at, &map_a, kb * 128, tm * 256 + rank * 128, b);
                        tma_load_2d_pair(at + Cfg::A_BYTES, &map_b, kb * 128, tn * BN + rank * Cfg::B_ROWS, b);
                    } else {
                        const uint32_t b = bar(Cfg::FULL + s);
                        mbar_expect(b, a.bytes);
                        tma_load_2d(at, &map_a, kb * 128, tm * 128, b);
                        tma_load_2d(at + Cfg::A_BYTES, &map_b, kb * 128, tn * BN, b);
                    }
                }
                __syncwarp();
            }
        }
        if constexpr (PAIR)   // nor an arrival of the products', which the pair's first CTA sends to both
            for (int i = max(0, it - STAGES); ok && i < it; ++i) ok = tc_wait(bar(Cfg::EMPTY + i % STAGES), (uint32_t)(i / STAGES) & 1u, abort_flag, a.status, 70);
        // No copy may arrive once the CTA has gone: where a wait gave up, the ones under way are waited for here (bounded like every wait; those of a pair
        // by its first CTA, and neither leaves before the other).
        if (rank == 0 && (!ok || *abort_flag))
            for (int i = max(0, it - STAGES); i < it; ++i) {
                int spins = 0;
                while (!tc_mbar_try(bar(Cfg::FULL + i % STAGES), (uint32_t)(i / STAGES) & 1u))
                    if (++spins > TC_WAIT_LIMIT) break;
            }
    } else if (warp == 1) {   // products, by the first CTA of a pair for both
        int it = 0, t = 0;
        bool ok = rank == 0;
        for (int tile = unit; ok && tile < tiles; tile += units, ++t) {
            const int acc = t % ACCS;
            if (t >= ACCS && !(ok = PAIR ? tc_wait_pair<false>(bar(Cfg::READ + acc), (uint32_t)(t / ACCS - 1) & 1u, abort_flag, a.status, 71)
                                      : tc_wait(bar(Cfg::READ + acc), (uint32_t)(t / ACCS - 1) & 1u, abort_flag, a.status, 71)))
                break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int kb = 0; kb < a.kblocks; ++kb, ++it) {
                const int s = it % STAGES;
                if (!(ok = PAIR ? tc_wait_pair<true>(bar(Cfg::FULL + s), (uint32_t)(it / STAGES) & 1u, abort_flag, a.status, 72)
                                : tc_wait(bar(Cfg::FULL + s), (uint32_t)(it / STAGES) & 1u, abort_flag, a.status, 72)))
                    break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (tc_elect()) {
                    const uint64_t da = tc_b_desc(smem0 + (uint32_t)s * Cfg::STAGE), db = tc_b_desc(smem0 + (uint32_t)s * Cfg::STAGE + Cfg::A_BYTES);
                    const int steps = kb + 1 == a.kblocks ? a.last_steps : 4;
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        if (ks < steps) gi_mma<PAIR>(tmem + (uint32_t)(acc * BN), da + 2u * ks, db + 2u * ks, Cfg::IDESC, kb > 0 || ks > 0);
                    tc_commit<PAIR>(bar(Cfg::EMPTY + s));
                    if (kb + 1 == a.kblocks) tc_commit<PAIR>(bar(Cfg::DONE + acc));
                }
                __syncwarp();
            }
        }
        if (rank == 0 && (!ok || *abort_flag))   // products under way read shared memory and write tensor memory
            for (int i = max(0, it - STAGES); i < it; ++i) {
                int spins = 0;
                while (!tc_mbar_try(bar(Cfg::EMPTY + i % STAGES), (uint32_t)(i / STAGES) & 1u))
                    if (++spins > TC_WAIT_LIMIT) break;
            }
    } else {   // outputs: two warps per quarter of the accumulator's lanes, half of the columns each
        constexpr int COLS = GI_PIECE / sizeof(T), HALF = BN / 2;
        static_assert(HALF % COLS == 0 && COLS <= 32, "pieces of half a tile's rows");
        const int e = warp - 2, quarter = warp & 3, half = e >> 2;
        unsigned char* const boxes = smem + Cfg::OFF_OUT + e * Cfg::BOXES * GI_BOX;
        int turn = 0;
        float* const chan = reinterpret_cast<float*>(smem + Cfg::OFF_SCALE) + e * BN;
        // A tile's scales and biases are fetched a tile ahead.
        float sa[4] = {}, s[HALF / 32] = {}, bias[HALF / 32] = {};   // (of a lane's four rows; of its columns)
        int64_t row0 = 0, first = 0;
        const auto fetch_scales = [&](int tile) {
            int tm, tn;
            tc_tile(tile, a.m_tiles, a.n_tiles, tm, tn);
            row0 = (int64_t)tm * (128 * CTAS) + rank * 128 + quarter * 32, first = (int64_t)tn * BN + half * HALF;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t row = row0 + 8 * r + (lane >> 2);
                sa[r] = row < a.m ? a.a_scale[row] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < HALF / 32; ++u) {
                const int64_t c = first + u * 32 + lane;
                s[u] = c < a.n ? __ldg(a.b_scale + c) : 0.0f;
                bias[u] = a.bias && c < a.n ? __ldg(a.bias + c) : 0.0f;
            }
        };
        int t = 0;
        if (unit < tiles) fetch_scales(unit);
        for (int tile = unit; tile < tiles; tile += units, ++t) {
            const int acc = t % ACCS;
            const int64_t to_row = row0, to_col = first;
            uint64_t sa2[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) asm("mov.b64 %0, {%1, %1};" : "=l"(sa2[r]) : "f"(sa[r]));
            __syncwarp();
#pragma unroll
            for (int u = 0; u < HALF / 32; ++u) chan[gi_place<T>(u * 32 + lane)] = s[u], chan[HALF + gi_place<T>(u * 32 + lane)] = bias[u];
            __syncwarp();
            if (tile + units < tiles) fetch_scales(tile + units);
            if (a.kblocks > 0 && !(PAIR ? tc_wait_pair<false>(bar(Cfg::DONE + acc), (uint32_t)(t / ACCS) & 1u, abort_flag, a.status, 73)
                                        : tc_wait(bar(Cfg::DONE + acc), (uint32_t)(t / ACCS) & 1u, abort_flag, a.status, 73)))
                break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at = tmem + (uint32_t)(acc * BN + half * HALF) + ((uint32_t)quarter << 21);
            const int cols = to_row >= a.m ? 0 : (int)min((int64_t)HALF, a.n - to_col);   // (the same for the warp)
            uint32_t v[2][COLS] = {};
            if (cols > 0 && a.kblocks > 0) gi_fetch<T>(at, v[0]);
#pragma unroll
            for (int c = 0; c < HALF; c += COLS) {
                if (c >= cols) break;
                uint32_t(&now)[COLS] = v[c / COLS & 1];
                tc_wait_loads(now);
                if (c + COLS < cols && a.kblocks > 0) gi_fetch<T>(at + (uint32_t)(c + COLS), v[~(c / COLS) & 1]);
                // the copy that last read this box has done so: of the groups since then, one a piece, as many may be under way as there are other boxes
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(Cfg::BOXES - 1) : "memory");
                __syncwarp();
                gi_write<T, HALF>(a, &map_c, boxes + turn * GI_BOX, chan + c, to_row, to_col + c, sa2, now);
                turn = (turn + 1) % Cfg::BOXES;
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (lane == 0) {
                if constexpr (PAIR) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(tc_pair_first(bar(Cfg::READ + acc))) : "memory");
                else tc_mbar_arrive(bar(Cfg::READ + acc));
            }
            __syncwarp();
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (PAIR) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // (the other one's arrivals and copies)
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1) {
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::TM_COLS) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::TM_COLS) : "memory");
    }
}

template <typename T, int BN, bool PAIR> int gi_launch(s2v_ctx* ctx, cudaStream_t st, const s2v_gemm_i8_args& g, bool dependent)
{
    using Cfg = GiCfg<BN, PAIR>;
    constexpr int ROWS = PAIR ? 256 : 128;
    // (a box with many rows outside the matrix takes longer than a full one: 27 rows of 128, 22 us instead of 16)
    const int box_a = (int)(g.m < 128 ? g.m : 128), box_b = (int)(g.n < Cfg::B_ROWS ? g.n : Cfg::B_ROWS);
    CUtensorMap map_a, map_b, map_c;
    if (g.k > 0) {
        // (the leading dimension of a single row is not the caller's to get right)
        const int64_t up = (g.k + 15) / 16 * 16;
        if (!s2v_byte_matrix_map(&map_a, g.A, g.m, g.k, g.m > 1 ? g.lda : up, box_a) || !s2v_byte_matrix_map(&map_b, g.B, g.n, g.k, g.n > 1 ? g.ldb : up, box_b))
            return s2v_fail(ctx, S2V_ERR_CUDA, "gemm_i8: the driver did not take a matrix's tensor map");
    } else {
        memset(&map_a, 0, sizeof(map_a));
        memset(&map_b, 0, sizeof(map_b));
    }
    GiArgs a;
    a.m = g.m, a.n = g.n, a.ldc = g.ldc;
    a.kblocks = (int)((g.k + 127) / 128);
    a.last_steps = g.k > 0 ? (int)((g.k - 128 * (int64_t)(a.kblocks - 1) + 31) / 32) : 0;
    const int64_t mt = (g.m + ROWS - 1) / ROWS, nt = (g.n + BN - 1) / BN;
    if (mt * nt > INT32_MAX / 2) return s2v_fail(ctx, S2V_ERR_UNSUPPORTED, "gemm_i8: more than 2^30 tiles of outputs");
    a.m_tiles = (int)mt, a.n_tiles = (int)nt, a.bytes = (uint32_t)(box_a + box_b) * 128;
    a.a_scale = g.a_scale, a.b_scale = g.b_scale, a.bias = g.bias, a.C = g.C, a.relu = g.relu;
    const int64_t es = sizeof(T), ldc = g.m > 1 ? g.ldc : (g.n * es + 15) / 16 * 16 / es;
    a.boxes = s2v_aligned16(g.C) && ldc * es % 16 == 0;
    if (!a.boxes) memset(&map_c, 0, sizeof(map_c));
    else if (!s2v_output_map(&map_c, g.c_type, g.C, g.m, g.n, ldc)) return s2v_fail(ctx, S2V_ERR_CUDA, "gemm_i8: the driver did not take the output's tensor map");
    a.status = ctx->dstatus_dev;
    S2V_CUDA_OK(ctx, s2v_allow_shared(gemm_i8_kernel<T, BN, PAIR>, Cfg::SMEM));
    const int64_t tiles = mt * nt, units = ctx->sm_count / (PAIR ? 2 : 1);
    const unsigned grid = (unsigned)(tiles < units ? tiles : units) * (PAIR ? 2 : 1);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(GI_THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIR ? 2 : 1;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 2 : 1;
    S2V_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, gemm_i8_kernel<T, BN, PAIR>, map_a, map_b, map_c, a));
    S2V_CHECK_LAUNCH(ctx, "gemm_i8_kernel");
    return S2V_OK;
}

// What a call takes by each form, in us, fitted to times of 148 SMs (16-bit outputs, every form at k = 128 to 14336, n = 256 to 14336, m = 16 to
// 20000; mostly within 15 %): `fixed` with the first tile's outputs, `first` and `next` for 128 columns of k in the first and in further tiles of a CTA
// (the further ones share L2 with everybody), `out` for a further tile's outputs where they take longer than that.  Measured sides of some choices:
//                          256 x 256 pair  256 x 128 pair  128 x 256  128 x 128  128 x 64   split
//     4096 x 4096 x 4096        46              63             58         78        137                  (m x n x k)
//     1024 x 4096 x 4096        16.3            21.7           17.3       25.0       42.5
//      512 x 4096 x 4096        15.4            13.5           16.5       14.8       23.4       22
//      200 x  256 x 4096        14.6            12.2           15.7       13.8       12.7        8.1
//       64 x 4096 x  512         7.1             5.8            6.6        5.3        4.7        7.2
//       27 x 4096 x 4096        14.7            12.6           15.6       13.8       12.9        7.2
//     5000 x 4096 x 1024        20.1            27.8           23.7       31.0       51.1
//    20000 x 4096 x  128        47.6            54.5           44.2       52.6       65.3
struct GiForm {
    int rows, bn;
    float fixed, first, next, out;
};
constexpr GiForm GI_PAIR_256{256, 256, 5.6f, .35f, .305f, 2.55f}, GI_PAIR_128{256, 128, 5.3f, .258f, .268f, 1.42f}, GI_256{128, 256, 4.7f, .45f, .44f, 2.55f},
    GI_128{128, 128, 4.55f, .329f, .334f, 1.45f}, GI_64{128, 64, 4.2f, .255f, .333f, .89f};

float gi_cost(const s2v_ctx* ctx, const s2v_gemm_i8_args& g, const GiForm& f)
{
    const int64_t units = ctx->sm_count / (f.rows / 128);
    if (units == 0) return INFINITY;
    const float panels = (float)((g.k + 127) / 128), waves = (float)((((g.m + f.rows - 1) / f.rows) * ((g.n + f.bn - 1) / f.bn) + units - 1) / units);
    const float out = f.out * (g.c_type == S2V_F32 ? 1.45f : 1.0f), next = f.next * panels;
    return f.fixed + out - f.out + f.first * panels + (waves - 1.0f) * (out > next ? out : next);
}

}  // namespace

int s2v_launch_gemm_i8(s2v_ctx* ctx, cudaStream_t st, const s2v_gemm_i8_args& g, bool dependent)
{
    if (s2v_gemv_i8_takes(g.m, g.n, g.k)) return s2v_launch_gemv_i8(ctx, st, -1, g);
    const GiForm* best = &GI_64;
    float least = gi_cost(ctx, g, GI_64);
    for (const GiForm* f : {&GI_128, &GI_256, &GI_PAIR_128, &GI_PAIR_256})
        if (const float c = gi_cost(ctx, g, *f); g.k > 0 && c < least) best = f, least = c;
    if (g.k > 0 && s2v_gemm_i8_split_cost(ctx, g) < least) return s2v_launch_gemm_i8_split(ctx, st, g, dependent);
    return s2v_by_dtype(g.c_type, [&](auto type) {
        using T = decltype(type);
        return best == &GI_PAIR_256 ? gi_launch<T, 256, true>(ctx, st, g, dependent) : best == &GI_PAIR_128 ? gi_launch<T, 128, true>(ctx, st, g, dependent)
             : best == &GI_256      ? gi_launch<T, 256, false>(ctx, st, g, dependent) : best == &GI_128      ? gi_launch<T, 128, false>(ctx, st, g, dependent)
                                                                                                            : gi_launch<T, 64, false>(ctx, st, g, dependent);
    });
}
