// Thin wrappers over the tcgen05 (5th-generation tensor core) PTX used by the product and attention kernels: tensor
// memory, the matrix instructions, and mbarrier waits that end.
#pragma once
#include "common.cuh"

namespace qcc {

__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}

// Barriers by shared-memory address (32 bits: a kernel with many of them then keeps one base register, the rest are immediates)
__device__ __forceinline__ void mbar_init_at(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) { asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void sts_u32(uint32_t addr, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t lds_volatile(uint32_t addr)
{
    uint32_t v;
    asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
// Wait for phase `parity`: whether it was reached.  The wait is bounded: when it runs out it records `code` in the device error word and
// raises `abort` (shared memory), which makes every later wait of the CTA return soon, so that the kernel ends, with its tensor memory freed,
// and the host reads the error.  Who arms a barrier or issues copies or matrix instructions behind the wait has to leave where it was not:
// arming a barrier again whose phase is incomplete is undefined.
[[nodiscard]] __device__ __forceinline__ bool mbar_reached(uint32_t bar, uint32_t parity, unsigned int code, uint32_t abort)
{
    for (uint32_t it = 0; it < (1u << 22); it++) {
        uint32_t done;
        asm volatile(
            "{\n.reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if ((it & 63u) == 63u && lds_volatile(abort)) return false;
    }
    asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(abort), "r"(1u) : "memory");
    atomicMax(&g_qcc_error, code);
    return false;
}
// the same for who only reads what the phase brings, or looks at the abort word later
__device__ __forceinline__ void mbar_wait_at(uint32_t bar, uint32_t parity, unsigned int code, uint32_t abort) { (void)mbar_reached(bar, parity, code, abort); }

// The end of a kernel in which a wait has run out: copies and matrix instructions that are still under way get a millisecond to end
// before the CTA's shared and tensor memory are given up.  By all threads, after the last barrier of the CTA: by then nobody issues any more.
__device__ __forceinline__ void settle(uint32_t abort)
{
    if (lds_volatile(abort))
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
}

__device__ __forceinline__ void tma_load_2d_at(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}

// --------------------------------------------------------------------------------------------- tensor memory
// The address of `cols` columns (a power of two >= 32) lands in `slot` (shared memory).  One whole warp calls it.
__device__ __forceinline__ void tmem_alloc_at(uint32_t slot, uint32_t cols)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// arrives on `bar` once every matrix instruction issued by this thread so far has finished
__device__ __forceinline__ void tc_commit_at(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 32 lanes (of this warp's quadrant) x 32 columns of 32 bits: thread = lane, r[i] = column i
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
          "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}

}  // namespace qcc
