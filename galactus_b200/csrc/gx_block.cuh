// The norms around a block, one pass over the rows (sm_100a):
//
//   m    = sum over s of w[s] y[s]  +  sigmoid(g) shared
//   out  = residual + scale * gate * norm(m)
//   next = norm(out)
//
// with norm(v) = v / sqrt(mean(v^2) + eps) * weight. Every part may be absent;
// the norm before a block is `next` of a single row y.
#pragma once

#include "gx_gmm.cuh"

namespace gx {

constexpr int kBlockUnit = 8;                     // elements of a thread's step: 16 bytes of a 16-bit type
constexpr int kBlockUnits = 2;                    // steps that a thread keeps in registers
constexpr int kBlockMaxThreads = 512;
constexpr int kBlockMaxCluster = 8;
constexpr int kBlockMaxWidth = kBlockUnit * kBlockUnits * kBlockMaxThreads * kBlockMaxCluster;

struct BlockRows {           // rows of a matrix: base, bytes between rows, type (GMM_*); NULL: absent
    uint8_t * p;
    int64_t nb;
    int32_t type;
};

struct BlockParams {
    int32_t H, T, k;
    BlockRows y;              // row (t, s) at y.p + t * y_nb2 + s * y.nb
    int64_t y_nb2;
    const float * w;          // [T, k] or NULL
    const int32_t * ids;      // [T, k] or NULL: slots with a negative id are left out
    BlockRows shared;
    const float * shared_gate;   // [T] or NULL
    const float * norm;       // [H]
    int32_t has_norm, has_next;
    float eps, next_eps, scale;
    const float * gate;       // or NULL
    int64_t gate_nb;          // 0: one row for all
    int32_t gate_step;        // 1: a value per element; 0: one per row
    int32_t gate_sigmoid;
    BlockRows res, dst, next;
    const float * next_norm;  // [H] or NULL (ones)
};

// elements i .. i + 7 of a row (below n), as f32
template <bool VEC>
__device__ __forceinline__ void block_load(const uint8_t * row, int type, int i, int n, float (&v)[kBlockUnit]) {
    if (VEC) {
        if (type == GMM_F32) {
            const float4 a = *reinterpret_cast<const float4 *>(row + (int64_t)i * 4);
            const float4 b = *reinterpret_cast<const float4 *>(row + (int64_t)i * 4 + 16);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = *reinterpret_cast<const uint4 *>(row + (int64_t)i * 2);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (type == GMM_BF16) {
                    v[2 * j] = __uint_as_float(w[j] << 16);
                    v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
                } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
                    v[2 * j] = f.x;
                    v[2 * j + 1] = f.y;
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < kBlockUnit; ++j) {
            v[j] = 0.0f;
            if (i + j < n) {
                if (type == GMM_F32) v[j] = reinterpret_cast<const float *>(row)[i + j];
                else if (type == GMM_BF16) v[j] = __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(row)[i + j]);
                else v[j] = __half2float(reinterpret_cast<const __half *>(row)[i + j]);
            }
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void block_store(uint8_t * row, int type, int i, int n, const float (&v)[kBlockUnit]) {
    if (VEC) {
        if (type == GMM_F32) {
            *reinterpret_cast<float4 *>(row + (int64_t)i * 4) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4 *>(row + (int64_t)i * 4 + 16) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (type == GMM_BF16) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t *>(&b);
                } else {
                    const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t *>(&h);
                }
            }
            *reinterpret_cast<uint4 *>(row + (int64_t)i * 2) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kBlockUnit; ++j)
            if (i + j < n) store_out(row, i + j, v[j], type);
    }
}

// The sum of v over the row's threads: the warps of a CTA, then the CTAs of
// the row's cluster, each in their order. `warps`, `ctas`: buffers of this sum alone.
template <bool CLUSTER>
__device__ __forceinline__ float block_sum(float v, float * warps, float * ctas) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, d));
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    if (lane == 0) warps[warp] = v;
    __syncthreads();
    v = 0.0f;
    for (int i = 0; i < n; ++i) v = __fadd_rn(v, warps[i]);
    if constexpr (CLUSTER) {
        uint32_t me, size;
        asm("mov.u32 %0, %cluster_ctarank;" : "=r"(me));
        asm("mov.u32 %0, %cluster_nctarank;" : "=r"(size));
        if (threadIdx.x < size)
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(peer_addr(ctas + me, (int)threadIdx.x)), "f"(v) : "memory");
        cluster_sync_all();
        v = 0.0f;
        for (uint32_t i = 0; i < size; ++i) v = __fadd_rn(v, ctas[i]);
    }
    return v;
}

__device__ __forceinline__ float block_sigmoid(float g) { return __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-g))); }

// A CTA, or a cluster of them, per row of the result.
template <bool VEC, bool CLUSTER>
__global__ void __launch_bounds__(kBlockMaxThreads) k_block(const __grid_constant__ BlockParams p) {
    __shared__ float warps[2][kBlockMaxThreads / 32], ctas[2][kBlockMaxCluster];
    const int tid = threadIdx.x;
    int rank = 0, size = 1;
    if constexpr (CLUSTER) {
        asm("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %cluster_nctarank;" : "=r"(size));
    }
    const int t = (int)blockIdx.x / size;
    const int first = (rank * (int)blockDim.x + tid) * kBlockUnit, step = size * (int)blockDim.x * kBlockUnit;
    griddep_launch_dependents();
    if constexpr (CLUSTER) cluster_sync_all();      // (peers are written to once they run)
    griddep_wait();

    float m[kBlockUnits][kBlockUnit], r[kBlockUnits][kBlockUnit];
    float ss = 0.0f;
#pragma unroll
    for (int u = 0; u < kBlockUnits; ++u) {
        const int i = first + u * step;
#pragma unroll
        for (int j = 0; j < kBlockUnit; ++j) m[u][j] = r[u][j] = 0.0f;
        if (i >= p.H) continue;
        const uint8_t * row = p.y.p + (int64_t)t * p.y_nb2;
        if (p.w == nullptr && p.ids == nullptr && p.k == 1) {
            block_load<VEC>(row, p.y.type, i, p.H, m[u]);
        } else {
            // in slot order, a rounded product and a rounded add each
            for (int s = 0; s < p.k; ++s) {
                if (p.ids != nullptr && p.ids[(int64_t)t * p.k + s] < 0) continue;
                float v[kBlockUnit];
                block_load<VEC>(row + (int64_t)s * p.y.nb, p.y.type, i, p.H, v);
                const float w = p.w != nullptr ? p.w[(int64_t)t * p.k + s] : 1.0f;
#pragma unroll
                for (int j = 0; j < kBlockUnit; ++j) m[u][j] = __fadd_rn(m[u][j], __fmul_rn(w, v[j]));
            }
        }
        if (p.shared.p != nullptr) {
            float v[kBlockUnit];
            block_load<VEC>(p.shared.p + (int64_t)t * p.shared.nb, p.shared.type, i, p.H, v);
            const float w = p.shared_gate != nullptr ? block_sigmoid(p.shared_gate[t]) : 1.0f;
#pragma unroll
            for (int j = 0; j < kBlockUnit; ++j) m[u][j] = __fadd_rn(m[u][j], __fmul_rn(w, v[j]));
        }
        if (p.res.p != nullptr) block_load<VEC>(p.res.p + (int64_t)t * p.res.nb, p.res.type, i, p.H, r[u]);
#pragma unroll
        for (int j = 0; j < kBlockUnit; ++j) ss = __fmaf_rn(m[u][j], m[u][j], ss);
    }
    float inv = 1.0f;
    if (p.has_norm) {
        ss = block_sum<CLUSTER>(ss, warps[0], ctas[0]);
        inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)p.H), p.eps)));
    }
    float ss2 = 0.0f;
#pragma unroll
    for (int u = 0; u < kBlockUnits; ++u) {
        const int i = first + u * step;
        if (i >= p.H) continue;
        float v[kBlockUnit];
        if (p.has_norm) {
            if (p.norm != nullptr) {
                block_load<false>(reinterpret_cast<const uint8_t *>(p.norm), GMM_F32, i, p.H, v);
#pragma unroll
                for (int j = 0; j < kBlockUnit; ++j) m[u][j] = __fmul_rn(__fmul_rn(m[u][j], inv), v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < kBlockUnit; ++j) m[u][j] = __fmul_rn(m[u][j], inv);
            }
        }
        if (p.gate != nullptr) {
            const uint8_t * row = reinterpret_cast<const uint8_t *>(p.gate) + (int64_t)t * p.gate_nb;
            if (p.gate_step != 0) block_load<false>(row, GMM_F32, i, p.H, v);
            else
#pragma unroll
                for (int j = 0; j < kBlockUnit; ++j) v[j] = *reinterpret_cast<const float *>(row);
#pragma unroll
            for (int j = 0; j < kBlockUnit; ++j) m[u][j] = __fmul_rn(m[u][j], p.gate_sigmoid ? block_sigmoid(v[j]) : v[j]);
        }
#pragma unroll
        for (int j = 0; j < kBlockUnit; ++j) {
            m[u][j] = __fadd_rn(r[u][j], __fmul_rn(p.scale, m[u][j]));
            if (i + j < p.H) ss2 = __fmaf_rn(m[u][j], m[u][j], ss2);
        }
        if (p.dst.p != nullptr) block_store<VEC>(p.dst.p + (int64_t)t * p.dst.nb, p.dst.type, i, p.H, m[u]);
    }
    if (!p.has_next) return;
    ss2 = block_sum<CLUSTER>(ss2, warps[1], ctas[1]);
    inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss2, (float)p.H), p.next_eps)));
#pragma unroll
    for (int u = 0; u < kBlockUnits; ++u) {
        const int i = first + u * step;
        if (i >= p.H) continue;
        float v[kBlockUnit];
        if (p.next_norm != nullptr) {
            block_load<false>(reinterpret_cast<const uint8_t *>(p.next_norm), GMM_F32, i, p.H, v);
#pragma unroll
            for (int j = 0; j < kBlockUnit; ++j) m[u][j] = __fmul_rn(__fmul_rn(m[u][j], inv), v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < kBlockUnit; ++j) m[u][j] = __fmul_rn(m[u][j], inv);
        }
        block_store<VEC>(p.next.p + (int64_t)t * p.next.nb, p.next.type, i, p.H, m[u]);
    }
}

}  // namespace gx
