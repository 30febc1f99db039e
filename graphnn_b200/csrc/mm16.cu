// Products of 16-bit matrices with fp32 accumulators in tensor memory: tcgen05.mma on tiles of 256 x 256 by a pair of CTAs, or of 128 x 128 by one.
//
// A persistent CTA (pair) walks over tiles, or over shares of k of tiles where these are few.  One warp copies panels of 64 numbers along k into a ring of
// six stages (tensor maps, 128-byte swizzle; zeros outside the matrices), one issues the products, eight take finished accumulators out of tensor memory, of
// which there are two.  A matrix that lies along k is a panel of rows of 128 bytes; one that lies across k (the weights of dx = G W, both operands of
// dW = G^T x) is copied as it lies, 64 rows of k by 128 bytes, and read transposed by the matrix instructions, so nothing is transposed in memory.
//
// The matrix instructions cut what they add to an accumulator instead of rounding it: over a long k a sum comes out too small by half a step of fp32 an
// instruction (loss of a token over k = 4096: 4.7e-6 off, relative; 2.7e-7 with fp32 units).  So an accumulator takes MM_CHUNK panels only, and the
// epilogue warps, which would wait otherwise, add them up in registers, rounded.  The tensor cores go on with the next tile's first two accumulators while a tile's
// outputs leave: with four panels each that is too short for 256 x 256 of them (4096 x 131072 x 2048, sums: 1.81 ms; eight panels 1.70, sixteen 1.66).
//
// Tiles that are left over when every unit has had its last full turn are cut along k, so that all units share them; their parts' sums go through memory
// and a second kernel.
#include <algorithm>
#include <cstring>

#include "mm16.cuh"
#include "tcgen05_pair.cuh"
#include "tma.cuh"

namespace
{

constexpr int MM_EPI = 8;                      // epilogue warps, behind a warp of copies, one of products and two that do nothing
constexpr int MM_THREADS = 32 * (4 + MM_EPI);
// Registers of a thread at launch, all that 384 threads can have; of the first four warps and of the epilogue warps of pairs, which hold 128 columns of sums:
// 128 * (40 + 2 * 232) = 384 * 168.
constexpr int MM_REGS = 168;
constexpr int MM_K = 64;                       // numbers along k of a panel
constexpr int MM_CHUNK = 8, MM_CHUNK_16 = 32;   // panels that an accumulator takes; where the outputs are 16-bit numbers
constexpr int MM_PIECE = 64, MM_BOX = 32 * MM_PIECE, MM_BOXES = 2;   // bytes of an output row that an epilogue warp hands over at a time; of its 32 rows; boxes of a warp
constexpr uint32_t MM_BLOCK = 64 * 128;        // bytes of 64 rows of k by 64 numbers across

template <int BN, bool PAIR> struct MmCfg {
    static constexpr int ROWS = PAIR ? 256 : 128, B_ROWS = PAIR ? BN / 2 : BN;
    static constexpr uint32_t A_BYTES = 128 * 128, B_BYTES = B_ROWS * 128, STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = 6, ACCS = 2;
    static constexpr uint32_t TM_COLS = ACCS * BN;
    enum { FULL = 0, EMPTY = FULL + STAGES, DONE = EMPTY + STAGES, READ = DONE + ACCS, BARS = READ + ACCS };
    static constexpr uint32_t OFF_OUT = STAGES * STAGE, OFF_BAR = OFF_OUT + MM_EPI * MM_BOXES * MM_BOX, OFF_MISC = OFF_BAR + 8 * BARS, SMEM = OFF_MISC + 16 + 1024;   // + slack to align the base to 1024 bytes
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct MmArgs {
    int64_t m, n;
    int m_tiles, n_tiles;
    int full, rest, splits;             // tiles by one unit each; the others, and the shares of k of each of them
    int steps, per_split, chunk;        // panels of a tile, all parts' products; of a share; of an accumulator
    int products, last_mmas;            // products of parts; instructions of a panel at the end of k
    uint32_t a_parts, b_parts;          // four bits a product
    int a_boxes, b_boxes;               // boxes of an operand that lies across
    uint32_t bytes, idesc;
    const int32_t* target;
    const float* weight;
    int64_t vocab, first;
    float2* part;
    float* mine;
    const float2* stats;
    const float* row_scale;
    void* g;
    int64_t ldg, g_part;
    int g_type, g_parts;
    const float* alpha;
    int alpha_rows;
    float* sum;
    int64_t pitch;
    int add;
    float* lines;
    void* out;
    const float* fix;
    const void* fix_w;
    int64_t fix_ld;
    int fix_wide;                       // rows of fix_w lie on 16-byte boundaries
    int64_t ldo;
    int out_type, boxes;                // boxes: the output has a tensor map (rows on 16-byte boundaries)
    s2v_device_status* status;
};

template <bool PAIR> __device__ __forceinline__ void mm_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar)
{
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x), "r"(y),
                     "r"(z), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                     : "memory");
}

// ---- outputs: a row a lane, 32 columns at a time
__device__ __forceinline__ void mm_store32(void* p, const uint32_t* w)   // 32 bytes on a 32-byte boundary
{
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
// 2^x as the hardware has it (two steps off at most); NaN stays, -infinity gives 0
__device__ __forceinline__ float mm_exp2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
constexpr float MM_LOG2E = 1.4426950408889634f;

// the row's class, far below 0 if it is left out or behind the last row
__device__ __forceinline__ int64_t mm_own(const MmArgs& a, int64_t row)
{
    constexpr int64_t NONE = -((int64_t)1 << 40);
    if (row >= a.m) return NONE;
    const int64_t t = a.target[row];
    return t < 0 || t >= a.vocab || (a.weight && a.weight[row] == 0.0f) ? NONE : t;
}

// A row's largest output and the sum of exponentials relative to it, joined with 32 more outputs.
struct mm_sums {
    float m = -INFINITY, l = 0.0f;
    __device__ __forceinline__ void add(const float* v)
    {
        float top = m;
#pragma unroll
        for (int j = 0; j < 32; ++j) top = fmaxf(top, v[j]);
        const float from = top == -INFINITY ? 0.0f : top;   // (all excluded so far; of NaN alone fmaxf gives -infinity too, and they reach the sum below)
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j) s += mm_exp2((v[j] - from) * MM_LOG2E);
        l = fmaf(l, m == -INFINITY ? 0.0f : mm_exp2((m - from) * MM_LOG2E), s);
        m = top;
    }
};

// y += f times `cols` numbers of a row
template <typename T> __device__ __forceinline__ void mm_add_row(const T* p, float f, float* y, int cols, bool wide)
{
    constexpr int N = PIECE<T>;
#pragma unroll
    for (int c = 0; c < 32; c += N) {
        if (wide && c + N <= cols) {
            float w[N];
            unpack_piece(*reinterpret_cast<const uint4*>(p + c), w, T());
#pragma unroll
            for (int e = 0; e < N; ++e) y[c + e] = fmaf(f, w[e], y[c + e]);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (c + e < cols) y[c + e] = fmaf(f, to_f32(p[c + e]), y[c + e]);
        }
    }
}
// 32 outputs of each of the warp's 32 rows, a row a lane, as boxes of 64-byte rows whose 16-byte pieces are exchanged by the 64-byte swizzle (which keeps the
// stores free of bank conflicts), and from there by one copy, or, where rows don't lie on 16-byte boundaries, by 16 lanes a row.  (A lane's own stores along
// its row: 50021 x 1021 of fp16 over 1531 rows, rows at odd places, 569 us.)
template <typename T> __device__ __forceinline__ void mm_write(const MmArgs& a, const CUtensorMap* map, unsigned char* boxes, int& turn, int64_t row0, int64_t col, int n, const float* y)
{
    constexpr int COLS = MM_PIECE / sizeof(T), PER = 16 / sizeof(T);
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < 32; c += COLS) {
        if (c >= n) break;
        unsigned char* const box = boxes + turn * MM_BOX;
        turn = (turn + 1) % MM_BOXES;
        // the copy that last read this box has done so: of the groups since then, one a box, as many may be under way as there are other boxes
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(MM_BOXES - 1) : "memory");
        __syncwarp();
#pragma unroll
        for (int p = 0; p < 4; ++p) *reinterpret_cast<uint4*>(box + lane * MM_PIECE + 16 * (p ^ (lane >> 1 & 3))) = pack_piece(y + c + p * PER, T());
        // (a copy that meets the end of a row inside 16 bytes writes zeros behind it, into what may be somebody else's)
        if (a.boxes && (col + c + COLS <= a.n || a.n % PER == 0)) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tma_store_2d(map, (int)(col + c), (int)row0, smem_u32(box));
        } else {
            // A word of four bytes a lane, two rows at a time; in a row of 16-bit numbers at an odd place a lane writes the second half of its word with the first half of
            // its neighbour's, the first lane the first number and the last lane the last one.  Two rows on, a row lies as this one does, so that all of this is found once.
            // (Found for each row: 50021 x 1021 of fp16 over 1531 rows 252 us, as many outputs of 16 bytes 124.)
            __syncwarp();
            const int l = lane & 15, hi = lane >> 4;
            const int cols = (int)min((int64_t)COLS, a.n - col - c), rows = (int)min((int64_t)32, a.m - row0) - hi;
            T* const p = static_cast<T*>(a.out) + (row0 + hi) * a.ldo + col + c;
            const int64_t step = 2 * a.ldo;
            uint32_t at[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) at[i] = smem_u32(box) + (uint32_t)(hi * MM_PIECE + 16 * ((l >> 2) ^ i) + 4 * (l & 3));
            const auto word = [&](int i) {
                uint32_t w;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at[i & 3] + (uint32_t)(i * 2 * MM_PIECE)) : "memory");
                return w;
            };
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t w = word(i);
                    if (2 * i < rows && l < cols) *reinterpret_cast<uint32_t*>(p + l + i * step) = w;
                }
            } else {
                uint16_t* const h = reinterpret_cast<uint16_t*>(p) + 2 * l;
                const bool odd = reinterpret_cast<uintptr_t>(h) & 2;
                const bool both = odd ? l < 15 && 2 * l + 2 < cols : 2 * l + 1 < cols, low = odd ? l == 0 : 2 * l < cols && !both, high = odd && !both && 2 * l + 1 < cols;
                const uint32_t pick = odd ? 0x5432u : 0x3210u;
                uint16_t* const h2 = h + (odd ? 1 : 0);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t w = word(i), next = __shfl_down_sync(0xffffffffu, w, 1);
                    if (2 * i < rows) {
                        if (both) *reinterpret_cast<uint32_t*>(h2 + i * step) = __byte_perm(w, next, pick);
                        if (low) h[i * step] = (uint16_t)w;
                        if (high) h[1 + i * step] = (uint16_t)(w >> 16);
                    }
                }
            }
            // among copies a piece is a bulk group in any case: the wait before a box is filled counts groups, and this one's turn is over like a copy's
            if (a.boxes && lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            __syncwarp();
        }
    }
}

template <int KIND, int BN, bool PAIR>
__global__ void __launch_bounds__(MM_THREADS, 1) mm16_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_c, const MmArgs a)
{
    using Cfg = MmCfg<BN, PAIR>;
    constexpr int STAGES = Cfg::STAGES, ACCS = Cfg::ACCS, CTAS = PAIR ? 2 : 1;
    constexpr bool A_ACROSS = KIND == MM16_OUT_ACROSS, B_ACROSS = KIND == MM16_OUT || KIND == MM16_OUT_ACROSS, OUT = KIND >= MM16_OUT;
    extern __shared__ unsigned char mm_raw[];
    unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(mm_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t smem0 = smem_u32(smem);
    const auto bar = [&](int i) { return smem0 + Cfg::OFF_BAR + 8u * (uint32_t)i; };
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::OFF_MISC);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_MISC + 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int items = a.full + a.rest * a.splits;
    const int rank = PAIR ? (int)(blockIdx.x & 1) : 0, unit = (int)blockIdx.x / CTAS, units = (int)gridDim.x / CTAS;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) tc_mbar_init(bar(Cfg::FULL + i), 1), tc_mbar_init(bar(Cfg::EMPTY + i), 1);
        for (int i = 0; i < ACCS; ++i) tc_mbar_init(bar(Cfg::DONE + i), 1), tc_mbar_init(bar(Cfg::READ + i), MM_EPI * CTAS);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&map_a), tma_prefetch_map(&map_b);
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
    // an item: a tile and all of its panels, or a share [from, to) of them
    const auto item_of = [&](int item, int& tm, int& tn, int& from, int& to) {
        const int over = item - a.full, split = over < 0 ? 0 : over / a.rest;
        tc_tile(over < 0 ? item : a.full + over - split * a.rest, a.m_tiles, a.n_tiles, tm, tn);
        from = over < 0 ? 0 : split * a.per_split, to = over < 0 ? a.steps : min(a.steps, from + a.per_split);
    };

    if (warp < 4) {
    if constexpr (PAIR) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {   // copies
        int it = 0;
        bool ok = true;
        for (int item = unit; ok && item < items; item += units) {
            int tm, tn, from, to;
            item_of(item, tm, tn, from, to);
            const int row = tm * Cfg::ROWS + rank * 128, col = tn * BN + rank * Cfg::B_ROWS;
            int kb = from / a.products, p = from - kb * a.products;
            for (int step = from; step < to; ++step, ++it) {
                const int s = it % STAGES;
                if (it >= STAGES && !(ok = tc_wait(bar(Cfg::EMPTY + s), (uint32_t)(it / STAGES - 1) & 1u, abort_flag, a.status, 80))) break;
                if (tc_elect()) {
                    const uint32_t at_a = smem0 + (uint32_t)s * Cfg::STAGE, at_b = at_a + Cfg::A_BYTES;
                    const int pa = (int)(a.a_parts >> 4 * p) & 15, pb = (int)(a.b_parts >> 4 * p) & 15;
                    uint32_t b = bar(Cfg::FULL + s);   // both CTAs' copies count on the first one's barrier, where the products are issued
                    if (rank == 0) mbar_expect(b, (PAIR ? 2 : 1) * a.bytes);
                    if constexpr (PAIR) b = tc_pair_first(b);
                    if constexpr (A_ACROSS)
                        for (int i = 0; i < a.a_boxes; ++i) mm_load<PAIR>(at_a + (uint32_t)i * MM_BLOCK, &map_a, row + i * 64, kb * MM_K, pa, b);
                    else mm_load<PAIR>(at_a, &map_a, kb * MM_K, row, pa, b);
                    if constexpr (B_ACROSS)
                        for (int i = 0; i < a.b_boxes; ++i) mm_load<PAIR>(at_b + (uint32_t)i * MM_BLOCK, &map_b, col + i * 64, kb * MM_K, pb, b);
                    else mm_load<PAIR>(at_b, &map_b, kb * MM_K, col, pb, b);
                }
                __syncwarp();
                if (++p == a.products) p = 0, ++kb;
            }
        }
        if constexpr (PAIR)   // nor an arrival of the products', which the pair's first CTA sends to both
            for (int i = max(0, it - STAGES); ok && i < it; ++i) ok = tc_wait(bar(Cfg::EMPTY + i % STAGES), (uint32_t)(i / STAGES) & 1u, abort_flag, a.status, 80);
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
        for (int item = unit; ok && item < items; item += units) {
            int tm, tn, from, to;
            item_of(item, tm, tn, from, to);
            for (int step = from, acc = 0; step < to; ++step, ++it) {
                const int at = (step - from) & (a.chunk - 1);
                const bool first = at == 0, last = at + 1 == a.chunk || step + 1 == to;   // of an accumulator
                if (first) {
                    acc = t % ACCS;
                    if (t >= ACCS && !(ok = PAIR ? tc_wait_pair<false>(bar(Cfg::READ + acc), (uint32_t)(t / ACCS - 1) & 1u, abort_flag, a.status, 81)
                                                 : tc_wait(bar(Cfg::READ + acc), (uint32_t)(t / ACCS - 1) & 1u, abort_flag, a.status, 81)))
                        break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    ++t;
                }
                const int s = it % STAGES;
                if (!(ok = PAIR ? tc_wait_pair<true>(bar(Cfg::FULL + s), (uint32_t)(it / STAGES) & 1u, abort_flag, a.status, 82)
                                : tc_wait(bar(Cfg::FULL + s), (uint32_t)(it / STAGES) & 1u, abort_flag, a.status, 82)))
                    break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (tc_elect()) {
                    const uint32_t at_a = smem0 + (uint32_t)s * Cfg::STAGE, at_b = at_a + Cfg::A_BYTES;
                    // 16 numbers of k: 32 bytes of a row along k, 16 rows of 128 bytes across
                    constexpr uint32_t STEP_A = A_ACROSS ? 128u : 2u, STEP_B = B_ACROSS ? 128u : 2u;
                    const uint64_t da = A_ACROSS ? tc_desc_across<MM_BLOCK>(at_a) : tc_b_desc(at_a), db = B_ACROSS ? tc_desc_across<MM_BLOCK>(at_b) : tc_b_desc(at_b);
                    const int mmas = step + a.products >= a.steps ? a.last_mmas : 4;
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        if (ks < mmas) tc_mma_f16<PAIR>(tmem + (uint32_t)(acc * BN), da + STEP_A * ks, db + STEP_B * ks, a.idesc, !first || ks > 0);
                    tc_commit<PAIR>(bar(Cfg::EMPTY + s));
                    if (last) tc_commit<PAIR>(bar(Cfg::DONE + acc));
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
    }
    } else {   // outputs: two warps per quarter of the accumulator's lanes, half of the columns each
        if constexpr (PAIR) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        constexpr int HALF = BN / 2;
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        int t = 0, turn = 0;
        bool ok = true;
        for (int item = unit; ok && item < items; item += units) {
            int tm, tn, from, to;
            item_of(item, tm, tn, from, to);
            const int64_t row = (int64_t)tm * Cfg::ROWS + rank * 128 + quarter * 32 + lane, col0 = (int64_t)tn * BN + half * HALF;
            int64_t own_at = -1;   // column of the row's own class
            float w = 0.0f;
            float2 st = make_float2(0.0f, 0.0f);
            if constexpr (KIND == MM16_SUMS || KIND == MM16_SOFTMAX_GRAD) own_at = mm_own(a, row) - a.first;
            if constexpr (KIND == MM16_SOFTMAX_GRAD)
                if (row < a.m) w = a.row_scale[row], st = a.stats[row];
            const int64_t left = row - lane >= a.m ? 0 : a.n - col0;
            const int cols = left < 0 ? 0 : left < HALF ? (int)left : HALF;   // (the same for the warp)
            float y[HALF];
#pragma unroll
            for (int j = 0; j < HALF; ++j) y[j] = 0.0f;
            for (int step = from; step < to; step += a.chunk, ++t) {
                const int acc = t % ACCS;
                if (!(ok = PAIR ? tc_wait_pair<false>(bar(Cfg::DONE + acc), (uint32_t)(t / ACCS) & 1u, abort_flag, a.status, 83)
                                : tc_wait(bar(Cfg::DONE + acc), (uint32_t)(t / ACCS) & 1u, abort_flag, a.status, 83)))
                    break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = tmem + (uint32_t)(acc * BN + half * HALF) + ((uint32_t)quarter << 21);
                uint32_t v[2][16];
                if (cols > 0) tc_ld_cols16(at, v[0]);
#pragma unroll
                for (int c = 0; c < HALF; c += 16) {
                    if (c >= cols) break;
                    uint32_t(&now)[16] = v[c / 16 & 1];
                    tc_wait_loads(now);
                    if (c + 16 < cols) tc_ld_cols16(at + (uint32_t)(c + 16), v[~(c / 16) & 1]);
#pragma unroll
                    for (int j = 0; j < 16; j += 2)
                        asm("{\n\t.reg .b64 s, v;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tadd.rn.f32x2 s, s, v;\n\tmov.b64 {%0, %1}, s;\n\t}"
                            : "+f"(y[c + j]), "+f"(y[c + j + 1])
                            : "f"(__uint_as_float(now[j])), "f"(__uint_as_float(now[j + 1])));
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(tc_pair_first(bar(Cfg::READ + acc))) : "memory");
                    else tc_mbar_arrive(bar(Cfg::READ + acc));
                }
                __syncwarp();
            }
            if (!ok) break;
            mm_sums sums;
#pragma unroll
            for (int c = 0; c < HALF; c += 32) {
                if (c >= cols) break;
                float* const now = y + c;
                const int n = min(32, cols - c);
                const int mine = own_at >= col0 + c && own_at < col0 + c + 32 ? (int)(own_at - col0 - c) : -1;
                if constexpr (KIND == MM16_SUMS) {
                    if (n < 32) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (j >= n) now[j] = -INFINITY;
                    }
                    if (__any_sync(0xffffffffu, mine >= 0)) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (j == mine) a.mine[row] = now[j], now[j] = -INFINITY;
                    }
                    sums.add(now);
                } else if constexpr (KIND == MM16_SOFTMAX_GRAD) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) now[j] = w == 0.0f ? 0.0f : w * mm_exp2((now[j] - st.x) * MM_LOG2E);
                    if (__any_sync(0xffffffffu, mine >= 0)) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (j == mine) now[j] = w * st.y;
                    }
                    if (row < a.m) {   // (whole 64-byte pieces: what lies behind the last column is the row's own padding)
                        uint16_t* const to_g = static_cast<uint16_t*>(a.g) + row * a.ldg + col0 + c;
                        uint32_t h[16];
                        if (a.g_type == S2V_F16) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) h[j] = pack_16bit<__half>(now[2 * j], now[2 * j + 1]);
                            mm_store32(to_g, h), mm_store32(to_g + 16, h + 8);
                        } else
                            for (int p = 0; p < a.g_parts; ++p) {   // the nearest, then the nearest to what is left
#pragma unroll
                                for (int j = 0; j < 16; ++j) {
                                    h[j] = pack_16bit<__nv_bfloat16>(now[2 * j], now[2 * j + 1]);
                                    now[2 * j] -= __uint_as_float(h[j] << 16), now[2 * j + 1] -= __uint_as_float(h[j] & 0xffff0000u);
                                }
                                mm_store32(to_g + p * a.g_part, h), mm_store32(to_g + p * a.g_part + 16, h + 8);
                            }
                    }
                } else {
                    const bool whole = item < a.full;
                    if (whole) {
                        if (row < a.m) {
                            const float alpha = a.alpha ? a.alpha[a.alpha_rows ? row : 0] : 1.0f;
#pragma unroll
                            for (int j = 0; j < 32; ++j) now[j] *= alpha;
                            if (a.add) {
                                const float* const s = a.sum + row * a.pitch + col0 + c;
#pragma unroll
                                for (int j = 0; j < 32; j += 4)
                                    if (j < n) {
                                        const float4 f = *reinterpret_cast<const float4*>(s + j);   // (rows of a multiple of 8)
                                        now[j] += f.x, now[j + 1] += f.y, now[j + 2] += f.z, now[j + 3] += f.w;
                                    }
                            }
                            if (a.fix) {
                                const float f = a.fix[row];
                                if (f != 0.0f) {   // (of a row that is left out it is 0)
                                    const int64_t from_w = a.target[row] * a.fix_ld + col0 + c;
                                    if (a.out_type == S2V_F16) mm_add_row(static_cast<const __half*>(a.fix_w) + from_w, f, now, n, a.fix_wide);
                                    else mm_add_row(static_cast<const __nv_bfloat16*>(a.fix_w) + from_w, f, now, n, a.fix_wide);
                                }
                            }
                        }
                        if (a.out) {
                            unsigned char* const boxes = smem + Cfg::OFF_OUT + (warp - 4) * MM_BOXES * MM_BOX;
                            if (a.out_type == S2V_F32) mm_write<float>(a, &map_c, boxes, turn, row - lane, col0 + c, n, now);
                            else if (a.out_type == S2V_F16) mm_write<__half>(a, &map_c, boxes, turn, row - lane, col0 + c, n, now);
                            else mm_write<__nv_bfloat16>(a, &map_c, boxes, turn, row - lane, col0 + c, n, now);
                        }
                    }
                    if (row < a.m && (!whole || !a.out)) {
                        float* const s = whole ? a.sum + row * a.pitch + col0 + c
                                               : a.lines + ((int64_t)(item - a.full) * Cfg::ROWS + (rank * 128 + quarter * 32 + lane)) * BN + half * HALF + c;
#pragma unroll
                        for (int j = 0; j < 32; j += 8)
                            if (j < n) mm_store32(s + j, reinterpret_cast<const uint32_t*>(now + j));
                    }
                }
            }
            if constexpr (KIND == MM16_SUMS)
                if (row < a.m) a.part[(int64_t)(2 * tn + half) * a.m + row] = make_float2(sums.m, sums.l);
        }
        if (OUT && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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

// The tiles that were cut along k: out (or sum) = alpha * the shares' sums, added in their order (+ sum, and what fix gives)
template <int ROWS, int BN> __global__ void __launch_bounds__(256) mm16_lines_kernel(const MmArgs a)
{
    constexpr int PER_TILE = ROWS * BN / 4 / 256;   // CTAs
    const int over = (int)blockIdx.x / PER_TILE, at = ((int)blockIdx.x % PER_TILE * 256 + (int)threadIdx.x) * 4;
    int tm, tn;
    tc_tile(a.full + over, a.m_tiles, a.n_tiles, tm, tn);
    const int64_t row = (int64_t)tm * ROWS + at / BN, col = (int64_t)tn * BN + at % BN;
    if (row >= a.m || col >= a.n) return;
    const float* const from = a.lines + (int64_t)over * ROWS * BN + at;
    float y[4] = {};
    for (int s = 0; s < a.splits; ++s) {
        const float4 f = *reinterpret_cast<const float4*>(from + (int64_t)s * a.rest * ROWS * BN);
        y[0] += f.x, y[1] += f.y, y[2] += f.z, y[3] += f.w;
    }
    const float alpha = a.alpha ? a.alpha[a.alpha_rows ? row : 0] : 1.0f, fix = a.fix ? a.fix[row] : 0.0f;
    float* const s = a.sum + row * a.pitch + col;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (col + e >= a.n) break;
        y[e] = alpha * y[e] + (a.add ? s[e] : 0.0f);
        if (fix != 0.0f) {
            const int64_t w = a.target[row] * a.fix_ld + col + e;
            y[e] = fmaf(fix, a.out_type == S2V_F16 ? to_f32(static_cast<const __half*>(a.fix_w)[w]) : to_f32(static_cast<const __nv_bfloat16*>(a.fix_w)[w]), y[e]);
        }
        const int64_t to = row * a.ldo + col + e;
        if (!a.out) s[e] = y[e];
        else if (a.out_type == S2V_F32) static_cast<float*>(a.out)[to] = y[e];
        else if (a.out_type == S2V_F16) static_cast<__half*>(a.out)[to] = from_f32<__half>(y[e]);
        else static_cast<__nv_bfloat16*>(a.out)[to] = from_f32<__nv_bfloat16>(y[e]);
    }
}

// ---- 16-bit parts of a matrix: eight columns a thread
template <typename T, bool WIDE, int PARTS>
__global__ void __launch_bounds__(256) mm16_pack_kernel(int64_t rows, int64_t cols, const T* __restrict__ x, int64_t ldx, const int32_t* __restrict__ target, const float* __restrict__ weight,
                                                        int64_t vocab, uint16_t* __restrict__ out, int64_t ldo, int64_t part)
{
    const int64_t per_row = (cols + 7) / 8, all = rows * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row, col = (i - row * per_row) * 8;
        bool keep = true;
        if (target) {
            const int64_t t = target[row];
            keep = t >= 0 && t < vocab && !(weight && weight[row] == 0.0f);
        }
        const T* const from = x + row * ldx + col;
        uint16_t* const to = out + row * ldo + col;
        if constexpr (PARTS == 1) {   // 16-bit numbers as they are
            uint4 v = make_uint4(0, 0, 0, 0);
            if (keep) {
                if (WIDE && col + 8 <= cols) v = *reinterpret_cast<const uint4*>(from);
                else {
                    uint32_t h[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) h[e] = col + e < cols ? reinterpret_cast<const uint16_t*>(from)[e] : 0u;
                    v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
                }
            }
            *reinterpret_cast<uint4*>(to) = v;
        } else {
            float f[8];
            if (WIDE && col + 8 <= cols) {
                const float4 u = reinterpret_cast<const float4*>(from)[0], w = reinterpret_cast<const float4*>(from)[1];
                f[0] = u.x, f[1] = u.y, f[2] = u.z, f[3] = u.w, f[4] = w.x, f[5] = w.y, f[6] = w.z, f[7] = w.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = col + e < cols ? to_f32(from[e]) : 0.0f;
            }
            if (!keep) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = 0.0f;
            }
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                uint32_t h[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    h[j] = mm16_head(f[2 * j], f[2 * j + 1]);
                    f[2 * j] -= __uint_as_float(h[j] << 16), f[2 * j + 1] -= __uint_as_float(h[j] & 0xffff0000u);
                }
                *reinterpret_cast<uint4*>(to + p * part) = make_uint4(h[0], h[1], h[2], h[3]);
            }
        }
    }
}

bool mm_map(CUtensorMap* map, const mm16_operand& o, int box_rows)
{
    const auto encode = s2v_tensor_map_encoder();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.parts};
    const int64_t up = (o.cols + 7) / 8 * 8, ld = o.rows > 1 ? o.ld : up;   // (the leading dimension of a single row is not the caller's to get right)
    const cuuint64_t strides[2] = {(cuuint64_t)(ld * 2), (cuuint64_t)((o.parts > 1 ? o.part : ld) * 2)};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(o.p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int mm_products(const mm16_args& a) { return a.a.parts == 1 ? (a.b.parts == 1 ? 1 : 3) : a.b.parts == 1 ? 3 : 6; }

// Whether pairs of CTAs on tiles of 256 x 256: both matrices more than half of a tile, and half of the pairs busy, or enough panels to share out among them.
bool mm_pairs(const s2v_ctx* ctx, int64_t m, int64_t n, int64_t steps)
{
    const int64_t pairs = ctx->sm_count / 2, tiles = ((m + 255) / 256) * ((n + 255) / 256);
    return pairs > 0 && m > 128 && n > 128 && (tiles * 2 >= pairs || tiles * steps >= 32 * pairs);
}
// How the tiles are shared out: the last, incomplete turn in `splits` shares of k each, none below 16 panels (8 where there is no other turn).
struct MmShares {
    int64_t full, rest, splits;
    MmShares(int64_t units, int64_t tiles, int64_t steps)
    {
        rest = tiles % units, full = tiles - rest, splits = 1;
        if (rest) splits = std::min(units / rest, steps / (full ? 16 : 8));
        if (splits < 2) full = tiles, rest = 0, splits = 1;
    }
};
int64_t mm_steps(const mm16_args& a) { return (a.k + MM_K - 1) / MM_K * mm_products(a); }

template <int KIND, int BN, bool PAIR> int mm_launch(s2v_ctx* ctx, cudaStream_t st, const mm16_args& g)
{
    using Cfg = MmCfg<BN, PAIR>;
    constexpr bool A_ACROSS = KIND == MM16_OUT_ACROSS, B_ACROSS = KIND == MM16_OUT || KIND == MM16_OUT_ACROSS, OUT = KIND >= MM16_OUT;
    const auto boxes = [](int64_t rows) { return rows <= 64 ? 1 : rows <= 128 ? 2 : 4; };
    // (a box with many rows outside the matrix takes longer than a full one)
    const int box_a = A_ACROSS ? 64 : (int)(g.m < 128 ? g.m : 128), box_b = B_ACROSS ? 64 : (int)(g.n < Cfg::B_ROWS ? g.n : Cfg::B_ROWS);
    CUtensorMap map_a, map_b;
    if (!mm_map(&map_a, g.a, box_a) || !mm_map(&map_b, g.b, box_b)) return s2v_fail(ctx, S2V_ERR_CUDA, "the driver did not take a matrix's tensor map");
    MmArgs a = {};
    a.m = g.m, a.n = g.n;
    const int64_t mt = (g.m + Cfg::ROWS - 1) / Cfg::ROWS, nt = (g.n + BN - 1) / BN;
    if (mt * nt > INT32_MAX / 2) return s2v_fail(ctx, S2V_ERR_UNSUPPORTED, "more than 2^30 tiles of outputs");
    a.m_tiles = (int)mt, a.n_tiles = (int)nt;
    const int64_t kblocks = (g.k + MM_K - 1) / MM_K;
    a.products = mm_products(g);
    // small parts first would gain nothing: the accumulator holds a rounding of its own size either way
    a.a_parts = g.a.parts == 1 ? 0u : g.b.parts == 1 ? 0x210u : 0x201100u;
    a.b_parts = g.b.parts == 1 ? 0u : g.a.parts == 1 ? 0x210u : 0x021010u;
    if (kblocks * a.products > INT32_MAX / 2) return s2v_fail(ctx, S2V_ERR_UNSUPPORTED, "more than 2^30 panels of k");
    a.steps = (int)kblocks * a.products;
    const int64_t units = std::min(ctx->sm_count, 148) / (PAIR ? 2 : 1);
    MmShares shares(units, mt * nt, a.steps);
    if (!OUT) shares.full = mt * nt, shares.rest = 0, shares.splits = 1;
    a.full = (int)shares.full, a.rest = (int)shares.rest;
    a.per_split = (int)((a.steps + shares.splits - 1) / shares.splits);
    a.splits = (a.steps + a.per_split - 1) / a.per_split;
    a.chunk = KIND == MM16_SUMS || a.products > 1 || (OUT && g.out_type == S2V_F32) ? MM_CHUNK : MM_CHUNK_16;
    a.last_mmas = (int)((g.k - MM_K * (kblocks - 1) + 15) / 16);
    a.a_boxes = A_ACROSS ? boxes(PAIR || g.m > 128 ? 128 : g.m) : 0, a.b_boxes = B_ACROSS ? boxes(PAIR || g.n > 128 ? 128 : g.n) : 0;
    a.bytes = (A_ACROSS ? (uint32_t)a.a_boxes * MM_BLOCK : (uint32_t)box_a * 128) + (B_ACROSS ? (uint32_t)a.b_boxes * MM_BLOCK : (uint32_t)box_b * 128);
    const uint32_t type = g.type == S2V_BF16 ? 1u : 0u;
    a.idesc = (1u << 4) | (type << 7) | (type << 10) | ((A_ACROSS ? 1u : 0u) << 15) | ((B_ACROSS ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(Cfg::ROWS >> 4) << 24);
    a.target = g.target, a.weight = g.weight, a.vocab = g.vocab, a.first = g.first;
    a.part = g.part, a.mine = g.mine, a.stats = g.stats, a.row_scale = g.row_scale;
    a.g = g.g, a.ldg = g.ldg, a.g_part = g.g_part, a.g_type = g.type, a.g_parts = g.g_parts;
    a.alpha = g.alpha, a.alpha_rows = g.alpha_rows, a.sum = g.sum, a.pitch = mm16_pitch(g.n), a.add = g.add, a.lines = g.lines;
    a.out = g.out, a.ldo = g.ldo, a.out_type = g.out_type;
    CUtensorMap map_c;
    const int64_t es = (int64_t)s2v_dtype_bytes(g.out_type), ldo = g.m > 1 ? g.ldo : (g.n * es + 15) / 16 * 16 / es;
    a.boxes = g.out && s2v_aligned16(g.out) && ldo * es % 16 == 0;
    if (!a.boxes) memset(&map_c, 0, sizeof(map_c));
    else if (!s2v_output_map(&map_c, g.out_type, g.out, g.m, g.n, ldo)) return s2v_fail(ctx, S2V_ERR_CUDA, "the driver did not take the output's tensor map");
    a.fix = g.fix, a.fix_w = g.fix_w, a.fix_ld = g.vocab > 1 ? g.fix_ld : 0;
    a.fix_wide = s2v_aligned16(g.fix_w) && (g.vocab <= 1 || g.fix_ld % 8 == 0);
    a.status = ctx->dstatus_dev;
    S2V_CUDA_OK(ctx, s2v_allow_shared(mm16_kernel<KIND, BN, PAIR>, Cfg::SMEM));
    if (PAIR) {   // the epilogue warps would wait for good for registers that the block does not have
        static const int regs = [] {
            cudaFuncAttributes f;
            return cudaFuncGetAttributes(&f, mm16_kernel<KIND, BN, PAIR>) == cudaSuccess ? f.numRegs : 0;
        }();
        if (regs != MM_REGS) return s2v_fail(ctx, S2V_ERR_CUDA, "mm16_kernel was not compiled for the registers that it shares out");
    }
    const int64_t items = a.full + (int64_t)a.rest * a.splits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items < units ? items : units) * (PAIR ? 2 : 1));
    cfg.blockDim = dim3(MM_THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PAIR ? 2 : 1;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    S2V_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, mm16_kernel<KIND, BN, PAIR>, map_a, map_b, map_c, a));
    S2V_CHECK_LAUNCH(ctx, "mm16_kernel");
    if (a.rest) {
        mm16_lines_kernel<Cfg::ROWS, BN><<<(unsigned)(a.rest * (Cfg::ROWS * BN / 4 / 256)), 256, 0, st>>>(a);
        S2V_CHECK_LAUNCH(ctx, "mm16_lines_kernel");
    }
    return S2V_OK;
}

}  // namespace

int mm16_sum_lines(const s2v_ctx* ctx, int64_t m, int64_t n)
{
    const int64_t bn = mm_pairs(ctx, m, n, 0) ? 256 : 128;
    return (int)(2 * ((n + bn - 1) / bn));
}
int64_t mm16_sum_lines_most(int64_t n) { return 2 * ((n + 127) / 128); }

size_t mm16_lines_bytes(int64_t k, int products)
{
    // a share of a tile of 256 x 256 for each of 74 pairs (as much as of 128 x 128 for each of 148 CTAs, twice over); none where k is too short to be shared out
    return (k + MM_K - 1) / MM_K * products < 16 ? 0 : (size_t)74 * 256 * 256 * sizeof(float);
}

int mm16_launch(s2v_ctx* ctx, cudaStream_t st, mm16_kind kind, const mm16_args& a)
{
    if (a.m == 0 || a.n == 0) return S2V_OK;
    const bool pairs = mm_pairs(ctx, a.m, a.n, kind >= MM16_OUT ? mm_steps(a) : 0);
    switch (kind) {
        case MM16_SUMS: return pairs ? mm_launch<MM16_SUMS, 256, true>(ctx, st, a) : mm_launch<MM16_SUMS, 128, false>(ctx, st, a);
        case MM16_SOFTMAX_GRAD: return pairs ? mm_launch<MM16_SOFTMAX_GRAD, 256, true>(ctx, st, a) : mm_launch<MM16_SOFTMAX_GRAD, 128, false>(ctx, st, a);
        case MM16_OUT: return pairs ? mm_launch<MM16_OUT, 256, true>(ctx, st, a) : mm_launch<MM16_OUT, 128, false>(ctx, st, a);
        case MM16_OUT_ACROSS: return pairs ? mm_launch<MM16_OUT_ACROSS, 256, true>(ctx, st, a) : mm_launch<MM16_OUT_ACROSS, 128, false>(ctx, st, a);
        default: return pairs ? mm_launch<MM16_OUT_ALONG, 256, true>(ctx, st, a) : mm_launch<MM16_OUT_ALONG, 128, false>(ctx, st, a);
    }
}

int mm16_pack(s2v_ctx* ctx, cudaStream_t st, int64_t rows, int64_t cols, int x_type, const void* x, int64_t ldx, const int32_t* target, const float* weight, int64_t vocab, void* out,
              int64_t ldo, int64_t part)
{
    const int64_t blocks = (rows * ((cols + 7) / 8) + 255) / 256, cap = 32 * (int64_t)ctx->sm_count;
    if (blocks == 0) return S2V_OK;
    const bool wide = s2v_aligned16(x) && (rows <= 1 || ldx * (int64_t)s2v_dtype_bytes(x_type) % 16 == 0);
    const auto go = [&](auto kernel, auto* from) {
        kernel<<<(unsigned)(blocks < cap ? blocks : cap), 256, 0, st>>>(rows, cols, from, ldx, target, weight, vocab, static_cast<uint16_t*>(out), ldo, part);
        S2V_CHECK_LAUNCH(ctx, "mm16_pack_kernel");
        return (int)S2V_OK;
    };
    if (x_type == S2V_F32) return wide ? go(mm16_pack_kernel<float, true, 3>, static_cast<const float*>(x)) : go(mm16_pack_kernel<float, false, 3>, static_cast<const float*>(x));
    return wide ? go(mm16_pack_kernel<__half, true, 1>, static_cast<const __half*>(x)) : go(mm16_pack_kernel<__half, false, 1>, static_cast<const __half*>(x));
}
