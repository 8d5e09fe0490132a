// Host-side helpers of the entry points: argument checks, launch limits of the
// current device, tensor maps of 16-bit rows.
#pragma once

#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <cstdio>

#include "../../include/galactus_b200.h"
#include "gx_gmm.cuh"

namespace {

int cuda_status(cudaError_t e) {
    if (e == cudaSuccess) return GX_OK;
    std::fprintf(stderr, "galactus_b200: CUDA error: %s\n", cudaGetErrorString(e));
    return e == cudaErrorMemoryAllocation ? GX_ERR_NOMEM : GX_ERR_CUDA;
}

constexpr int kMaxDevices = 64;

// multiprocessors of the current device
int device_sms() {
    static std::atomic<int> sms[kMaxDevices];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
    if ((n = sms[dev].load(std::memory_order_relaxed)) == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        sms[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// kernels of one source file that need more dynamic shared memory than a launch has by default
constexpr int kKernelSlots = 32;

// Lets `fn` have up to `bytes` on the current device: the most that any call
// asks for, set once. (The limit belongs to the function, not to a call. One
// set to each call's own size would let another thread's smaller call lower it
// before the launch.)
cudaError_t allow_smem(const void * fn, int slot, uint32_t bytes) {
    static std::atomic<bool> done[kMaxDevices][kKernelSlots];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    if (done[dev][slot].load(std::memory_order_acquire)) return cudaSuccess;
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done[dev][slot].store(true, std::memory_order_release);
    return e;
}

// Clusters of a kernel that run at once (SMs are grouped in GPCs of unequal
// size, so clusters of 4 or 8 leave some out), one CTA per SM. The kernel has
// been given its shared memory (allow_smem); `slot` names it in the table of
// what was asked before.
int resident_clusters(const void * fn, int cluster, int threads, uint32_t smem, int slot) {
    static std::atomic<int> known[kMaxDevices][kKernelSlots][4];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
    std::atomic<int> & k = known[dev][slot][cluster == 1 ? 0 : cluster == 2 ? 1 : cluster == 4 ? 2 : 3];
    int n = k.load(std::memory_order_relaxed);
    if (n > 0) return n;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)cluster);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess || n <= 0) return 0;
    k.store(n, std::memory_order_relaxed);
    return n;
}

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void * f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    return fn;
}

// rows of K 16-bit elements, boxes of `width` (16, 32, 64) elements by `box`
// rows, swizzled over the width
bool encode_rows(CUtensorMap * map, bool bf16, const void * base, int64_t K, int64_t rows, int64_t nb1, int64_t mats,
                 int64_t nb2, uint32_t box, uint32_t width = gx::kGmmK) {
    const auto enc = map_encoder();
    if (enc == nullptr) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)rows, (cuuint64_t)mats};
    const cuuint64_t strides[2] = {(cuuint64_t)nb1, (cuuint64_t)nb2};
    const cuuint32_t boxes[3] = {width, box, 1u};
    const cuuint32_t elem[3] = {1u, 1u, 1u};
    return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, mats > 0 ? 3 : 2,
               const_cast<void *>(base), dims, strides, boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
               width == 64u   ? CU_TENSOR_MAP_SWIZZLE_128B
               : width == 32u ? CU_TENSOR_MAP_SWIZZLE_64B
                              : CU_TENSOR_MAP_SWIZZLE_32B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool misaligned(const void * p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// whether `rows` rows `pitch` bytes apart, `last` bytes of the last one, fit in `stride` bytes
bool rows_fit(int64_t rows, int64_t pitch, int64_t last, int64_t stride) {
    return (__int128)(rows - 1) * pitch + last <= stride;
}

int out_kind(int type) {
    return type == GX_TYPE_F32 ? gx::GMM_F32 : type == GX_TYPE_F16 ? gx::GMM_F16 : type == GX_TYPE_BF16 ? gx::GMM_BF16 : -1;
}

// Whether one accumulator is too short for sums of K elements. The tensor
// cores' f32 accumulators drop what does not fit instead of rounding: for
// products of random signs about 1e-9 of the magnitudes' sum per element, for
// products of one sign 6e-9 (measured: 4.8e-5 at K = 7168, 1.6e-4 at 28672).
// Results of 16 bits do not see that while it is a fifth of half a step.
bool long_sum(int out, int64_t K) { return K > (out == gx::GMM_F32 ? 512 : out == gx::GMM_F16 ? 16384 : 131072); }

constexpr int64_t kMaxIndex = 0x7fffffff;
constexpr int64_t kMaxSize = kMaxIndex - 65536;      // of rows and elements: the kernels look a tile ahead in 32 bits
constexpr int64_t kMaxStride = 1ll << 40;      // of a tensor map

}  // namespace
