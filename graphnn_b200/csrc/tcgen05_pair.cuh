// What kernels share whose tiles a CTA or a pair of CTAs multiplies: commits and waits of a pair, products of 16-bit operands, the order of tiles, loads of accumulators.
#pragma once

#include "tcgen05.cuh"

namespace
{

// the barrier of this CTA, or of both of the pair, once all products issued so far are done
template <bool PAIR> __device__ __forceinline__ void tc_commit(uint32_t bar)
{
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// tc_wait for barriers on which the other CTA of the pair arrives too.  Where all that a barrier orders is accumulators in tensor memory, which tcgen05.fence
// takes care of, its arrivals and waits are relaxed (released and acquired at the cluster's scope they cost pairs of 256 x 128 a third of their time at
// k = 128, and a microsecond of 18 at 200 x 14336 x 4096).
template <bool ACQUIRE> __device__ __forceinline__ bool tc_wait_pair(uint32_t bar, uint32_t parity, volatile int* abort_flag, s2v_device_status* status, int site)
{
    int spins = 0;
    bool ok = true;
    for (;;) {
        uint32_t done;
        if constexpr (ACQUIRE)
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(done)
                         : "r"(bar), "r"(parity), "r"(TC_SUSPEND_NS)
                         : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(done)
                         : "r"(bar), "r"(parity), "r"(TC_SUSPEND_NS)
                         : "memory");
        if (done) break;
        if (*abort_flag) { ok = false; break; }
        if (++spins > TC_WAIT_LIMIT) {
            *abort_flag = 1;
            status->code = S2V_ERR_DEVICE_TIMEOUT;
            status->where = site;
            ok = false;
            break;
        }
    }
    return __all_sync(0xffffffffu, ok);
}
// the address of a barrier in the pair's first CTA
__device__ __forceinline__ uint32_t tc_pair_first(uint32_t bar)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(bar));
    return r;
}

// 16 numbers along k of 16-bit operands, by a CTA or by a pair, of which the first issues them for both.
template <bool PAIR> __device__ __forceinline__ void tc_mma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            :
            : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            :
            : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
}
// shared-memory descriptor of an operand across k: blocks of 64 numbers BLOCK bytes apart, in them 8 rows of k every 1024 bytes (128-byte swizzle)
template <uint32_t BLOCK> __device__ __forceinline__ uint64_t tc_desc_across(uint32_t smem_addr)
{
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3fffu);
    d |= (uint64_t)(BLOCK >> 4) << 16;      // leading byte offset: the next 64 numbers
    d |= (uint64_t)(1024 >> 4) << 32;       // stride byte offset: the next 8 rows of k
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// Tiles in columns of 16 row tiles, so that the tiles of one moment share panels of both matrices in L2.
__device__ __forceinline__ void tc_tile(int tile, int m_tiles, int n_tiles, int& tm, int& tn)
{
    constexpr int G = 16;
    const int per = G * n_tiles, g = tile / per, first = g * G, rows = min(G, m_tiles - first), at = tile - g * per;
    tm = first + at % rows;
    tn = at / rows;
}

// Accumulators that tcgen05.ld was asked for: no use of them comes before the wait.
template <int N> __device__ __forceinline__ void tc_wait_loads(uint32_t (&v)[N])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int j = 0; j < N; j += 8)
        asm volatile("" : "+r"(v[j]), "+r"(v[j + 1]), "+r"(v[j + 2]), "+r"(v[j + 3]), "+r"(v[j + 4]), "+r"(v[j + 5]), "+r"(v[j + 6]), "+r"(v[j + 7]));
}

}  // namespace
