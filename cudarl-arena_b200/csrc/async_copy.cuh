// async_copy.cuh -- asynchronous copies into shared memory, completion on an mbarrier, and bounded waits for it.
#pragma once
#include <cuda_runtime.h>

namespace cudarl {

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned long long* bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(smem_u32(bar)), "r"(count) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(unsigned long long* bar, unsigned bytes) {
    // relaxed: the barrier only tells this warp that its tensor copy has landed; no write of the arriving lane is published by it
    asm volatile("mbarrier.arrive.expect_tx.relaxed.cta.shared::cta.b64 _, [%0], %1;" :: "r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// The same by a lane that has written to shared memory itself what the barrier's waiters read.
__device__ __forceinline__ void mbar_publish_expect_tx(unsigned long long* bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" :: "r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned long long* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(smem_u32(bar)) : "memory"); }
// One look at the barrier, no waiting.
__device__ __forceinline__ bool mbar_test_wait(unsigned long long* bar, unsigned parity) {
    unsigned ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0u;
}
// Sleeps in hardware until the phase completes or about `ns` nanoseconds have passed: a waiting warp issues nothing.
__device__ __forceinline__ bool mbar_try_wait(unsigned long long* bar, unsigned parity, unsigned ns) {
    unsigned ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(ns) : "memory");
    return ok != 0u;
}
__device__ __forceinline__ void bulk_g2s(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ unsigned long long global_ns() {
    unsigned long long t; asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t)); return t;
}
constexpr unsigned long long WAIT_NS = 2000000000ull;   // a copy that has not landed after two seconds never will

// Wait for the phase with the given parity.  Bounded: by `polls` tries when polls > 0 (tests make a wait run
// out that way), else by WAIT_NS of wall time.  false = gave up.
__device__ __forceinline__ bool mbar_wait(unsigned long long* bar, unsigned parity, unsigned polls) {
    if (polls) {
        for (unsigned it = 0; it < polls; ++it) if (mbar_test_wait(bar, parity)) return true;
        return false;
    }
    unsigned long long t0 = 0ull;
    for (unsigned it = 1u;; ++it) {
        if (mbar_try_wait(bar, parity, 20000u)) return true;
        if ((it & 15u) == 0u) {
            const unsigned long long now = global_ns();
            if (t0 == 0ull) t0 = now; else if (now - t0 > WAIT_NS) return false;
        }
    }
}

}  // namespace cudarl
