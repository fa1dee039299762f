// mbarriers with bounded waits and the tcgen05 instructions that the products on the tensor cores share (dense.cu, rows8_mm.cu).
#pragma once

#include "pspmm_common.cuh"

namespace tc {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint32_t bar, int count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, int parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 0x989680;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// False when the wait ran out (or another role's did: *abort), which *status then tells.  Whole warps call it, and its lanes agree: what
// follows are barriers and tcgen05 instructions of whole warps.
__device__ __forceinline__ bool bar_wait(uint32_t bar, int parity, volatile int *abort, uint32_t limit_ns,
                                         unsigned *status)
{
    if (__all_sync(PSPMM_FULL_MASK, bar_try(bar, parity)))
        return true;
    unsigned long long t0, t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    while (!__all_sync(PSPMM_FULL_MASK, bar_try(bar, parity))) {
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
        if (__any_sync(PSPMM_FULL_MASK, *abort || t - t0 > limit_ns)) {
            *abort = 1;
            atomicExch(status, 1u);
            return false;
        }
    }
    return true;
}

__device__ __forceinline__ bool elect_one()
{
    uint32_t on;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
    return on != 0;
}
__device__ __forceinline__ void mma_commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// Eight accumulator columns of the warp's 32 TMEM lanes; complete after tcgen05.wait::ld.
__device__ __forceinline__ void acc_load(uint32_t (&v)[8], uint32_t addr)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(addr));
}

}  // namespace tc
