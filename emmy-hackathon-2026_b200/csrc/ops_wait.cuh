/* Waits on barriers in shared memory that end: each gives up after a limit. */
#pragma once

#include <stdint.h>

static constexpr uint64_t TIMEOUT_NS = 2000000000ull;

static __device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

static __device__ __forceinline__ bool try_wait(uint32_t barrier, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred q;\nmbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2;\nselp.u32 %0, 1, 0, q;\n}"
                 : "=r"(ok) : "r"(barrier), "r"(parity) : "memory");
    return ok;
}
static __device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
/* False when the wait gave up, here or in another role: after `limit` ns it sets *abort (of the block of threads) and the role's
 * bit in *status.  The timer is looked at in every 64th try only: most waits are for one block's product, and reading it is
 * slow. */
static __device__ __forceinline__ bool wait_for(uint32_t barrier, uint32_t parity, volatile unsigned *abort, unsigned *status, unsigned role,
                                                   uint64_t limit = TIMEOUT_NS) {
    uint64_t start = 0;
    for (unsigned tries = 0; !try_wait(barrier, parity); ++tries) {
        if ((tries & 63) != 63) continue;
        if (*abort) return false;
        const uint64_t now = now_ns();
        if (!start) start = now;
        if (now - start > limit) {
            *abort = 1;
            atomicOr(status, role);
            return false;
        }
    }
    return true;
}

/* both barriers, tried together first: a try takes tens of cycles, and one thread issues all products */
static __device__ __forceinline__ bool wait_for_both(uint32_t a, uint32_t a_parity, uint32_t b, uint32_t b_parity, volatile unsigned *abort,
                                                     unsigned *status, unsigned role, uint64_t limit = TIMEOUT_NS) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p, q;\n"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
                 "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n"
                 "and.pred p, p, q;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(a), "r"(a_parity), "r"(b), "r"(b_parity) : "memory");
    return ok || (wait_for(a, a_parity, abort, status, role, limit) && wait_for(b, b_parity, abort, status, role, limit));
}

/* Of one's own work under way, after a wait gave up: until it is done or the limit has passed since `start`. */
static __device__ __forceinline__ void wait_for_end(uint32_t barrier, uint32_t parity, uint64_t start, uint64_t limit = TIMEOUT_NS) {
    while (!try_wait(barrier, parity) && now_ns() - start < limit) {}
}
