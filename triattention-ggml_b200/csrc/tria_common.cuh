/*
 * tria_common.cuh - what the library's kernels share: the status bits, the
 * checked build's bounds test, and mbarriers with bounded waits.
 */
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <climits>

#include "tria_internal.h"

namespace tria {

enum : int { KT_F32SPLIT = 0, KT_F16 = TRIA_TYPE_F16, KT_Q8_0 = TRIA_TYPE_Q8_0 };
/* Bits of the device status word (tria_ctx's d_status), decoded on the host
 * by tria_status_of_bits(): a key position outside the table, a bounded
 * pipeline wait that gave up, a row count or an accepted path (both device
 * data) that does not fit its cache. */
enum : int { ST_POSITION = 1, ST_TIMEOUT = 2, ST_BOUNDS = 4, ST_ROWS = 8 };

/* Bounds checks of the checked build (compiled with TRIA_CHECKS): a failed
 * check sets ST_BOUNDS in *status and the caller skips the access.  In the
 * product build the check is the constant true and compiles away. */
__device__ __forceinline__ uint32_t dynamic_smem_bytes() {
    uint32_t b;
    asm("mov.u32 %0, %%dynamic_smem_size;" : "=r"(b));
    return b;
}
__device__ __forceinline__ bool bounds_ok(bool ok, int32_t *status) {
#ifdef TRIA_CHECKS
    if (!ok && status) atomicOr(status, ST_BOUNDS);
    return ok;
#else
    (void)ok;
    (void)status;
    return true;
#endif
}

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive_tx(uint64_t *bar, uint32_t bytes) {
    uint64_t st;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 %0, [%1], %2;"
                 : "=l"(st) : "r"(smem_u32(bar)), "r"(bytes) : "memory");
    asm volatile("" ::"l"(st));
}
__device__ __forceinline__ void mbar_expect(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    uint64_t st;
    asm volatile("mbarrier.arrive.shared::cta.b64 %0, [%1];" : "=l"(st) : "r"(smem_u32(bar)) : "memory");
    asm volatile("" ::"l"(st));
}
/* Non-multicast bulk copy global -> this CTA's shared memory. */
__device__ __forceinline__ void bulk_g2s(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
/* Non-blocking test of a phase (test_wait never suspends the thread). */
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
/* Default bound of a pipeline wait: ~2^31 cycles, about a second. */
constexpr long long WAIT_LIMIT_DEFAULT = 1ll << 31;
/* Wait for a phase of `bar`, giving up after `limit` cycles.  try_wait may
 * suspend the thread until the phase completes, which is the cheap way to
 * wait but can outlast a short bound; a bound shortened below the default
 * (the timeout-path test hook) polls with test_wait instead, so it is
 * checked every few dozen cycles. */
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, long long limit = WAIT_LIMIT_DEFAULT) {
    if (limit < WAIT_LIMIT_DEFAULT) {
        const long long t0 = clock64();
        while (!mbar_test(bar, parity))
            if (clock64() - t0 > limit) return false;
        return true;
    }
    if (mbar_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try(bar, parity))
        if (clock64() - t0 > limit) return false;
    return true;
}

}  // namespace tria
