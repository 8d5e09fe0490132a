// Bounded waits of the kernels that work in roles (products on grouped rows, with
// 4-bit weights, adapters, rings of rows). A wait that runs out is recorded
// (GX_DEVERR_TIMEOUT) and ends the other waits of its CTA; what the kernel writes
// from there on is NaN or nothing, and it leaves once its copies have landed.
#pragma once

#include "gx_device.cuh"

namespace gx {

__device__ __forceinline__ uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// one poll of a phase, with what the peer CTA's arrivals released (suspends for a while)
template <int CTAS>
__device__ __forceinline__ bool gmm_poll(uint64_t * bar, uint32_t parity) {
    if constexpr (CTAS == 1) return mbar_try_wait(bar, parity);
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, "
        "p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

// Bounded wait of a thread: gives up after two seconds, or once another role of the CTA has.
template <int CTAS>
__device__ __noinline__ bool gmm_wait_long(uint64_t * bar, uint32_t parity, volatile int * abort_flag) {
    uint64_t t0 = 0;
    for (uint32_t i = 1;; ++i) {
        if (gmm_poll<CTAS>(bar, parity)) return true;
        if ((i & 63u) == 0u) {
            if (*abort_flag != 0) return false;
            const uint64_t t = global_ns();
            if (t0 == 0) t0 = t;
            else if (t - t0 > 2000000000ull) {
                *abort_flag = 1;
                record_error(GX_DEVERR_TIMEOUT);
                return false;
            }
        }
    }
}
template <int CTAS>
__device__ __forceinline__ bool gmm_wait_one(uint64_t * bar, uint32_t parity, volatile int * abort_flag) {
    return gmm_poll<CTAS>(bar, parity) || gmm_wait_long<CTAS>(bar, parity, abort_flag);
}
// the same by a whole warp
template <int CTAS>
__device__ __forceinline__ bool gmm_wait(uint64_t * bar, uint32_t parity, volatile int * abort_flag) {
    return __all_sync(0xffffffffu, gmm_wait_one<CTAS>(bar, parity, abort_flag));
}

}  // namespace gx
