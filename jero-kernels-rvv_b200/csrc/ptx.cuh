// PTX wrappers shared by the kernels that wait on mbarriers or use the tensor core's own memory:
// bounded mbarrier waits, tcgen05 fences and commits, shared-memory operand descriptors and
// packed f32 pairs.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace jkb {

constexpr unsigned long long WAIT_NS = 2000000000ull;  // bounded waits: 2 s

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ unsigned long long globaltimer() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void mbar_init(uint64_t *b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count));
}
__device__ __forceinline__ bool mbar_try(uint64_t *b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Waits for the phase of parity `parity` to complete; false after WAIT_NS (which sets `bit` in the
// device error word) or when another role has aborted.
__device__ __forceinline__ bool mbar_wait_slow(uint64_t *b, uint32_t parity, volatile int *abort_flag,
                                               int *err, int bit = 1) {
    const unsigned long long t0 = globaltimer();
    for (uint32_t i = 1;; i++) {
        if (mbar_try(b, parity)) return true;
        if ((i & 255) == 0) {
            if (*abort_flag) return false;
            if (globaltimer() - t0 > WAIT_NS) {
                *abort_flag = 1;
                atomicOr(err, bit);
                return false;
            }
        }
    }
}
__device__ __forceinline__ bool mbar_wait(uint64_t *b, uint32_t parity, volatile int *abort_flag,
                                          int *err, int bit = 1) {
    return mbar_try(b, parity) || mbar_wait_slow(b, parity, abort_flag, err, bit);
}
// Bounded like mbar_wait_slow, with a short sleep between polls: for warps that run ahead of
// the MMA and would otherwise take issue slots from the epilogue warps.
__device__ __forceinline__ bool mbar_wait_sleepy(uint64_t *b, uint32_t parity,
                                                 volatile int *abort_flag, int *err) {
    if (mbar_try(b, parity)) return true;
    const unsigned long long t0 = globaltimer();
    for (;;) {
        __nanosleep(256);
        if (mbar_try(b, parity)) return true;
        if (*abort_flag) return false;
        if (globaltimer() - t0 > WAIT_NS) {
            *abort_flag = 1;
            atomicOr(err, 1);
            return false;
        }
    }
}
__device__ __forceinline__ void mbar_arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_tx(uint64_t *b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)),
                 "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t *b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     smem_u32(b))
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// K-major operand tile of 128-byte rows with the 128-byte swizzle: 8-row atoms 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(const void *p) {
    const uint64_t addr = smem_u32(p);
    return ((addr >> 4) & 0x3FFFull)           // start address
           | (1ull << 16)                      // leading byte offset (unused with swizzle)
           | ((uint64_t)(1024 >> 4) << 32)     // stride byte offset: next 8-row atom
           | (1ull << 46)                      // descriptor version (sm_100)
           | (2ull << 61);                     // SWIZZLE_128B
}
// Packed f32 pairs (two outputs per instruction).
__device__ __forceinline__ uint64_t pk2(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ void upk2(uint64_t v, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

}  // namespace jkb
