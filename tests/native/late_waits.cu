// The products with 4-bit weights and the norms around a block with a wait that
// runs out: the n-th wait of one warp is waited for as ever, then taken to have
// run out. Nothing is lost or late on the GPU, so every other role goes on as it
// would, and no wait takes its two seconds.
#include "gx_wait.cuh"

namespace gx {

struct LateWait {
    int block, warp, at, seen;
};
__device__ LateWait g_late = {-1, -1, -1, 0};

template <int CTAS>
__device__ bool late_wait(uint64_t * bar, uint32_t parity, volatile int * abort_flag) {
    bool ok = gmm_wait<CTAS>(bar, parity, abort_flag);
    if ((int)blockIdx.x == g_late.block && (int)(threadIdx.x >> 5) == g_late.warp) {
        int n = 0;
        if ((threadIdx.x & 31) == 0) n = atomicAdd(&g_late.seen, 1);
        if (__shfl_sync(0xffffffffu, n, 0) == g_late.at) {
            *abort_flag = 1;
            record_error(GX_DEVERR_TIMEOUT);
            ok = false;
        }
        __syncwarp();
    }
    return ok;
}

}  // namespace gx

#define gmm_wait late_wait
#include "gx_q4.cu"

extern "C" {

// the wait numbered `at` of a block's warp (none: -1); waits are counted from zero again
int late_set(int block, int warp, int at) {
    const gx::LateWait v{block, warp, at, 0};
    return (int)cudaMemcpyToSymbol(gx::g_late, &v, sizeof v);
}
// waits of that warp so far
int late_seen() {
    gx::LateWait v{};
    return cudaMemcpyFromSymbol(&v, gx::g_late, sizeof v) == cudaSuccess ? v.seen : -1;
}
int late_error() {
    int code = -1;
    return gx::read_and_clear_q4_error(&code) == cudaSuccess ? code : -1;
}

}  // extern "C"
