// The norms around a block, one pass over the rows (sm_100a):
//
//   m    = sum over s of w[s] y[s]  +  sigmoid(g) shared
//   out  = residual + scale * gate * norm(m)
//   next = norm(out)
//
// with norm(v) = v / sqrt(mean(v^2) + eps) * weight. Every part may be absent;
// the norm before a block is `next` of a single row y.
//
// Every row is read once and every result written once; what lies between stays in
// f32 registers (16 elements a thread). Two kernels:
//   k_block       narrow rows: a warp each, without a barrier (65536 rows of 128, sum,
//                 residual and next norm: 45 us, 109 with a CTA each). Others: a CTA per
//                 row, or a cluster of up to eight whose sums of squares are exchanged
//                 through their shared memories (wide rows, or so few wide rows that
//                 most SMs would idle): latency bound. One token:
//                 2.2 us (2880 elements, a norm), 3.4 us (2048 x 8 experts, with
//                 residual and next norm), of which a launch alone is about 2.
//   k_block_rows  many rows: HBM bound, as far as the instructions keep up. 8192 rows
//                 of 4096, f32 to bf16, a norm: 43 us, 4.7 TB/s; the sum over 8 experts,
//                 norm, gate, residual and next norm, bf16: 151 us, 5.8 TB/s (of 6.55
//                 measured for a copy); 517 rows of 7168, 37 % of the slots left out:
//                 32 us, 4.0 TB/s. One CTA per row took 65, 276 and 43 us: few loads
//                 are in flight, and rows wait for their sums.
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
    float one;                // 1 (see block_add)
    float per;                // 1 / H
    const float * gate;       // or NULL
    int64_t gate_nb;          // 0: one row for all
    int32_t gate_step;        // 1: a value per element; 0: one per row
    int32_t gate_sigmoid;
    BlockRows res, dst, next;
    const float * next_norm;  // [H] or NULL (ones)
};

// f32 pairs in 64-bit registers: two rounded operations per instruction
__device__ __forceinline__ uint64_t mul_x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
constexpr int kBlockPairs = kBlockUnit / 2;

// elements i .. i + 7 of a row (below n), as f32 pairs
template <bool VEC>
__device__ __forceinline__ void block_load(const uint8_t * row, int type, int i, int n, uint64_t (&v)[kBlockPairs]) {
    if (VEC) {
        if (type == GMM_F32) {
            const ulonglong2 a = *reinterpret_cast<const ulonglong2 *>(row + (int64_t)i * 4);
            const ulonglong2 b = *reinterpret_cast<const ulonglong2 *>(row + (int64_t)i * 4 + 16);
            v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
        } else {
            const uint4 a = *reinterpret_cast<const uint4 *>(row + (int64_t)i * 2);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < kBlockPairs; ++j) {
                if (type == GMM_BF16) v[j] = u2pack(w[j] << 16, w[j] & 0xFFFF0000u);
                else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
                    v[j] = f2pack(f.x, f.y);
                }
            }
        }
    } else {
        float f[kBlockUnit];
#pragma unroll
        for (int j = 0; j < kBlockUnit; ++j) {
            f[j] = 0.0f;
            if (i + j < n) {
                if (type == GMM_F32) f[j] = reinterpret_cast<const float *>(row)[i + j];
                else if (type == GMM_BF16) f[j] = __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(row)[i + j]);
                else f[j] = __half2float(reinterpret_cast<const __half *>(row)[i + j]);
            }
        }
#pragma unroll
        for (int j = 0; j < kBlockPairs; ++j) v[j] = f2pack(f[2 * j], f[2 * j + 1]);
    }
}

template <bool VEC>
__device__ __forceinline__ void block_store(uint8_t * row, int type, int i, int n, const uint64_t (&v)[kBlockPairs]) {
    if (VEC && type == GMM_F32) {
        *reinterpret_cast<ulonglong2 *>(row + (int64_t)i * 4) = make_ulonglong2(v[0], v[1]);
        *reinterpret_cast<ulonglong2 *>(row + (int64_t)i * 4 + 16) = make_ulonglong2(v[2], v[3]);
        return;
    }
    float f[kBlockUnit];
#pragma unroll
    for (int j = 0; j < kBlockPairs; ++j) f2unpack(v[j], f[2 * j], f[2 * j + 1]);
    if (VEC) {
        uint32_t w[kBlockPairs];
#pragma unroll
        for (int j = 0; j < kBlockPairs; ++j) {
            if (type == GMM_BF16) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t *>(&b);
            } else {
                const __half2 h = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        *reinterpret_cast<uint4 *>(row + (int64_t)i * 2) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int j = 0; j < kBlockUnit; ++j)
            if (i + j < n) store_out(row, i + j, f[j], type);
    }
}

// m += w v, a rounded product and a rounded add each. (`one` is 1, which the
// assembler does not know: it makes one operation, with one rounding, of a packed
// product and a packed sum.)
__device__ __forceinline__ void block_add(uint64_t (&m)[kBlockPairs], float w, const uint64_t (&v)[kBlockPairs], float one) {
    const uint64_t ww = f2pack(w, w), oo = f2pack(one, one);
#pragma unroll
    for (int j = 0; j < kBlockPairs; ++j) m[j] = fma_x2(mul_x2(ww, v[j]), oo, m[j]);
}
// m *= w (and v)
__device__ __forceinline__ void block_scale(uint64_t (&m)[kBlockPairs], float w) {
    const uint64_t ww = f2pack(w, w);
#pragma unroll
    for (int j = 0; j < kBlockPairs; ++j) m[j] = mul_x2(m[j], ww);
}
__device__ __forceinline__ void block_scale(uint64_t (&m)[kBlockPairs], const uint64_t (&v)[kBlockPairs]) {
#pragma unroll
    for (int j = 0; j < kBlockPairs; ++j) m[j] = mul_x2(m[j], v[j]);
}
// m = r + scale m
__device__ __forceinline__ void block_residual(uint64_t (&m)[kBlockPairs], float scale, const uint64_t (&r)[kBlockPairs]) {
    const uint64_t ww = f2pack(scale, scale);
#pragma unroll
    for (int j = 0; j < kBlockPairs; ++j) m[j] = fma_x2(ww, m[j], r[j]);
}
// the squares of m, added to a pair of sums
__device__ __forceinline__ uint64_t block_squares(const uint64_t (&m)[kBlockPairs], uint64_t ss) {
#pragma unroll
    for (int j = 0; j < kBlockPairs; ++j) ss = fma_x2(m[j], m[j], ss);
    return ss;
}
__device__ __forceinline__ float block_pair_sum(uint64_t v) {
    float a, b;
    f2unpack(v, a, b);
    return __fadd_rn(a, b);
}
// 1 / sqrt(ss / H + eps). CUDA's rsqrtf is within 2 steps of f32; a rounded root
// and quotient take 100 operations more, a quarter of a row's in the norm alone.
__device__ __forceinline__ float block_inverse_root(float ss, float per, float eps) { return rsqrtf(__fmaf_rn(ss, per, eps)); }
__device__ __forceinline__ float block_sigmoid(float g) { return __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-g))); }
// the gate of a row's elements i .. i + 7, times m
template <bool VEC>
__device__ __forceinline__ void block_gate(const BlockParams & p, int t, int i, uint64_t (&m)[kBlockPairs]) {
    const uint8_t * g = reinterpret_cast<const uint8_t *>(p.gate) + (int64_t)t * p.gate_nb;
    if (p.gate_step == 0) {
        const float v = *reinterpret_cast<const float *>(g);
        block_scale(m, p.gate_sigmoid ? block_sigmoid(v) : v);
        return;
    }
    uint64_t v[kBlockPairs];
    block_load<VEC>(g, GMM_F32, i, p.H, v);
    if (p.gate_sigmoid) {
#pragma unroll
        for (int j = 0; j < kBlockPairs; ++j) {
            float a, b;
            f2unpack(v[j], a, b);
            v[j] = f2pack(block_sigmoid(a), block_sigmoid(b));
        }
    }
    block_scale(m, v);
}

// what a row's elements are spread over
enum : int { ROW_WARP = 0, ROW_CTA = 1, ROW_CLUSTER = 2 };

// The sum of v over the row's threads: a warp, the warps of a CTA, then the CTAs
// of the row's cluster, each in their order. `warps`, `ctas`: buffers of this sum alone.
template <int OVER>
__device__ __forceinline__ float block_sum(float v, float * warps, float * ctas) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, d));
    if constexpr (OVER == ROW_WARP) return v;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    if (lane == 0) warps[warp] = v;
    __syncthreads();
    v = 0.0f;
    for (int i = 0; i < n; ++i) v = __fadd_rn(v, warps[i]);
    if constexpr (OVER == ROW_CLUSTER) {
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

constexpr int kBlockBatch = 4;      // rows of y that a thread loads before it adds them
constexpr int kBlockWarps = 8;      // rows of a CTA whose warps have one each
GX_HD constexpr int block_threads(int over) { return over == ROW_WARP ? 32 * kBlockWarps : kBlockMaxThreads; }

// A warp, a CTA, or a cluster of them, per row of the result.
template <int YT, bool VEC, int OVER, int kUnits>
__global__ void __launch_bounds__(block_threads(OVER)) k_block(const __grid_constant__ BlockParams p) {
    __shared__ float warps[2][kBlockMaxThreads / 32], ctas[2][kBlockMaxCluster];
    const int tid = threadIdx.x, lane = tid & 31;
    int rank = 0, size = 1;
    if constexpr (OVER == ROW_CLUSTER) {
        asm("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %cluster_nctarank;" : "=r"(size));
    }
    const int t = OVER == ROW_WARP ? (int)blockIdx.x * (int)(blockDim.x >> 5) + (tid >> 5) : (int)blockIdx.x / size;
    const int first = (OVER == ROW_WARP ? lane : rank * (int)blockDim.x + tid) * kBlockUnit;
    const int step = (OVER == ROW_WARP ? 32 : size * (int)blockDim.x) * kBlockUnit;
    griddep_launch_dependents();
    if constexpr (OVER == ROW_CLUSTER) cluster_sync_all();      // (peers are written to once they run)
    griddep_wait();
    if (OVER == ROW_WARP && t >= p.T) return;

    uint64_t m[kUnits][kBlockPairs], r[kUnits][kBlockPairs];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int i = first + u * step;
#pragma unroll
        for (int j = 0; j < kBlockPairs; ++j) m[u][j] = r[u][j] = 0ull;
        if (p.res.p != nullptr && i < p.H) block_load<VEC>(p.res.p + (int64_t)t * p.res.nb, p.res.type, i, p.H, r[u]);
    }
    const uint8_t * row = p.y.p + (int64_t)t * p.y_nb2;
    if (p.w == nullptr && p.ids == nullptr && p.k == 1) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int i = first + u * step;
            if (i < p.H) block_load<VEC>(row, YT, i, p.H, m[u]);
        }
    } else {
        // in slot order
        for (int s0 = 0; s0 < p.k; s0 += 32) {
            const int at = s0 + lane;
            const bool in = at < p.k && (p.ids == nullptr || p.ids[(int64_t)t * p.k + at] >= 0);
            const float wl = in && p.w != nullptr ? p.w[(int64_t)t * p.k + at] : 1.0f;
            const unsigned have = __ballot_sync(0xffffffffu, in);
            const int n = min(32, p.k - s0);
            for (int s = 0; s < n; s += kBlockBatch) {
#pragma unroll
                for (int u = 0; u < kUnits; ++u) {
                    const int i = first + u * step;
                    if (__all_sync(0xffffffffu, i >= p.H)) continue;
                    uint64_t v[kBlockBatch][kBlockPairs];
#pragma unroll
                    for (int b = 0; b < kBlockBatch; ++b)
                        if (i < p.H && s + b < n && (have >> (s + b) & 1u) != 0u)
                            block_load<VEC>(row + (int64_t)(s0 + s + b) * p.y.nb, YT, i, p.H, v[b]);
#pragma unroll
                    for (int b = 0; b < kBlockBatch; ++b) {
                        const float w = __shfl_sync(0xffffffffu, wl, (s + b) & 31);
                        if (i < p.H && s + b < n && (have >> (s + b) & 1u) != 0u) block_add(m[u], w, v[b], p.one);
                    }
                }
            }
        }
    }
    uint64_t ss = 0ull;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int i = first + u * step;
        if (i >= p.H) continue;
        if (p.shared.p != nullptr) {
            uint64_t v[kBlockPairs];
            block_load<VEC>(p.shared.p + (int64_t)t * p.shared.nb, p.shared.type, i, p.H, v);
            block_add(m[u], p.shared_gate != nullptr ? block_sigmoid(p.shared_gate[t]) : 1.0f, v, p.one);
        }
        ss = block_squares(m[u], ss);
    }
    float inv = 1.0f;
    if (p.has_norm) inv = block_inverse_root(block_sum<OVER>(block_pair_sum(ss), warps[0], ctas[0]), p.per, p.eps);
    ss = 0ull;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int i = first + u * step;
        if (i >= p.H) continue;
        uint64_t v[kBlockPairs];
        if (p.has_norm) {
            block_load<VEC>(reinterpret_cast<const uint8_t *>(p.norm), GMM_F32, i, p.H, v);
            block_scale(m[u], inv);
            block_scale(m[u], v);
        }
        if (p.gate != nullptr) block_gate<VEC>(p, t, i, m[u]);
        block_residual(m[u], p.scale, r[u]);
        ss = block_squares(m[u], ss);
        if (p.dst.p != nullptr) block_store<VEC>(p.dst.p + (int64_t)t * p.dst.nb, p.dst.type, i, p.H, m[u]);
    }
    if (!p.has_next) return;
    inv = block_inverse_root(block_sum<OVER>(block_pair_sum(ss), warps[1], ctas[1]), p.per, p.next_eps);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int i = first + u * step;
        if (i >= p.H) continue;
        block_scale(m[u], inv);
        if (p.next_norm != nullptr) {
            uint64_t v[kBlockPairs];
            block_load<VEC>(reinterpret_cast<const uint8_t *>(p.next_norm), GMM_F32, i, p.H, v);
            block_scale(m[u], v);
        }
        block_store<VEC>(p.next.p + (int64_t)t * p.next.nb, p.next.type, i, p.H, m[u]);
    }
}

// ------------------------------------------------------------ many rows

constexpr int kRowsMaxSlots = 32;
constexpr int kRowsMaxWarps = 16;                 // of them that compute
constexpr int kRowsMaxWidth = 32 * kRowsMaxWarps * kBlockUnit * kBlockUnits;

// CTAs per SM of up to `warps` computing warps
GX_HD constexpr int rows_ctas(int warps) { return warps <= 8 ? 3 : 1; }

// The same for many rows: persistent CTAs, one warp copies the rows of the
// tokens ahead into a ring of slots (one bulk copy a row), the others add them up
// as they arrive. p.k <= 32, aligned rows. (Packed f32 pairs halve the arithmetic;
// 2.6 instructions a cycle are issued in the sum over 8 experts.)
template <int YT, int MAXW>
__global__ void __launch_bounds__(32 * (MAXW + 1), rows_ctas(MAXW)) k_block_rows(const __grid_constant__ BlockParams p, int slots, int slot_bytes) {
    extern __shared__ __align__(128) uint8_t block_ring[];
    __shared__ uint64_t full[kRowsMaxSlots], empty[kRowsMaxSlots];
    __shared__ float sums[4][kRowsMaxWarps];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, W = (int)(blockDim.x >> 5) - 1;
    griddep_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < slots; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, (uint32_t)W);
        }
        abort_flag = 0;
        mbar_fence_init();
    }
    griddep_wait();
    __syncthreads();
    const int ysize = YT == GMM_F32 ? 4 : 2;
    // lane s: slot s of token t (its weight; whether it is there)
    auto slot_of = [&](int t, float & w) {
        const bool in = t < p.T && lane < p.k && (p.ids == nullptr || p.ids[(int64_t)t * p.k + lane] >= 0);
        w = in && p.w != nullptr ? p.w[(int64_t)t * p.k + lane] : 1.0f;
        return in;
    };
    RingPos at;
    bool ok = true;
    if (warp == W) {
        float none;
        bool in = slot_of((int)blockIdx.x, none);
        int issued = 0;
        auto copy = [&](const uint8_t * from, int bytes) {
            if (at.round != 0) ok = ok && gmm_wait<1>(empty + at.s, (at.round - 1u) & 1u, &abort_flag);
            if (!ok) return;
            if (elect_one()) {
                mbar_arrive_expect_tx(full + at.s, (uint32_t)bytes);
                bulk_g2s(block_ring + at.s * slot_bytes, from, (uint32_t)bytes, full + at.s);
            }
            __syncwarp();
            ++issued;
            at.next(slots);
        };
        for (int t = (int)blockIdx.x; t < p.T && ok; t += (int)gridDim.x) {
            unsigned have = __ballot_sync(0xffffffffu, in);
            in = slot_of(t + (int)gridDim.x, none);
            const uint8_t * row = p.y.p + (int64_t)t * p.y_nb2;
            for (; have != 0u; have &= have - 1u) copy(row + (int64_t)(__ffs((int)have) - 1) * p.y.nb, p.H * ysize);
            if (p.shared.p != nullptr) copy(p.shared.p + (int64_t)t * p.shared.nb, p.H * (p.shared.type == GMM_F32 ? 4 : 2));
            if (p.res.p != nullptr) copy(p.res.p + (int64_t)t * p.res.nb, p.H * (p.res.type == GMM_F32 ? 4 : 2));
        }
        // copies in flight land before the CTA leaves (those that compute may have given up on them)
        volatile int no_flag = 0;
        for (int i = 0; i < slots; ++i)
            if (issued > i) gmm_wait<1>(full + i, (uint32_t)((issued - 1 - i) / slots & 1), &no_flag);
        return;
    }

    const int first = tid * kBlockUnit, step = W * 32 * kBlockUnit;
    auto there = [&](int u) { return first + u * step < p.H; };
    uint64_t xw[kBlockUnits][kBlockPairs];
#pragma unroll
    for (int u = 0; u < kBlockUnits; ++u) {
#pragma unroll
        for (int j = 0; j < kBlockPairs; ++j) xw[u][j] = f2pack(1.0f, 1.0f);
        if (there(u) && p.next_norm != nullptr) block_load<true>(reinterpret_cast<const uint8_t *>(p.next_norm), GMM_F32, first + u * step, p.H, xw[u]);
    }
    // The next row of the ring, as f32. (A warp whose wait ran out hands no slot back: the
    // others then compute on what they have, and give up behind it.)
    auto take = [&](int type, uint64_t (&v)[kBlockUnits][kBlockPairs]) {
        ok = gmm_wait<1>(full + at.s, at.round & 1u, &abort_flag) && ok;
        const uint8_t * row = block_ring + at.s * slot_bytes;
#pragma unroll
        for (int u = 0; u < kBlockUnits; ++u)
            if (there(u)) block_load<true>(row, type, first + u * step, p.H, v[u]);
        __syncwarp();
        if (lane == 0 && ok) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(empty + at.s)) : "memory");
        at.next(slots);
    };
    auto sum = [&](float v, float * part) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, d));
        if (lane == 0) part[warp] = ok ? v : kNan;
        asm volatile("bar.sync 1, %0;" ::"r"(32 * W) : "memory");
        v = part[0];
        for (int i = 1; i < W; ++i) v = __fadd_rn(v, part[i]);
        return v;
    };
    float w_next;
    bool in_next = slot_of((int)blockIdx.x, w_next);
    int turn = 0;
    for (int t = (int)blockIdx.x; t < p.T; t += (int)gridDim.x, turn ^= 2) {
        const float wl = w_next;
        unsigned have = __ballot_sync(0xffffffffu, in_next);
        in_next = slot_of(t + (int)gridDim.x, w_next);
        float shared_w = 1.0f;
        if (p.shared_gate != nullptr) shared_w = p.shared_gate[t];
        uint64_t m[kBlockUnits][kBlockPairs], v[kBlockUnits][kBlockPairs];
#pragma unroll
        for (int u = 0; u < kBlockUnits; ++u)
#pragma unroll
            for (int j = 0; j < kBlockPairs; ++j) m[u][j] = v[u][j] = 0ull;
        // in slot order
        for (; have != 0u; have &= have - 1u) {
            take(YT, v);
            const float w = __shfl_sync(0xffffffffu, wl, __ffs((int)have) - 1);
#pragma unroll
            for (int u = 0; u < kBlockUnits; ++u) block_add(m[u], w, v[u], p.one);
        }
        if (p.shared.p != nullptr) {
            take(p.shared.type, v);
            const float w = p.shared_gate != nullptr ? block_sigmoid(shared_w) : 1.0f;
#pragma unroll
            for (int u = 0; u < kBlockUnits; ++u) block_add(m[u], w, v[u], p.one);
        }
        if (p.has_norm) {
            uint64_t ss = 0ull;
#pragma unroll
            for (int u = 0; u < kBlockUnits; ++u) ss = block_squares(m[u], ss);
            const float inv = block_inverse_root(sum(block_pair_sum(ss), sums[turn]), p.per, p.eps);
#pragma unroll
            for (int u = 0; u < kBlockUnits; ++u) {
                if (!there(u)) continue;
                uint64_t nw[kBlockPairs];
                block_load<true>(reinterpret_cast<const uint8_t *>(p.norm), GMM_F32, first + u * step, p.H, nw);
                block_scale(m[u], inv);
                block_scale(m[u], nw);
            }
        }
        if (p.gate != nullptr) {
#pragma unroll
            for (int u = 0; u < kBlockUnits; ++u)
                if (there(u)) block_gate<true>(p, t, first + u * step, m[u]);
        }
#pragma unroll
        for (int u = 0; u < kBlockUnits; ++u)
#pragma unroll
            for (int j = 0; j < kBlockPairs; ++j) v[u][j] = 0ull;
        if (p.res.p != nullptr) take(p.res.type, v);
        const float scale = ok ? p.scale : kNan;                     // (a wait ran out)
        uint64_t ss = 0ull;
#pragma unroll
        for (int u = 0; u < kBlockUnits; ++u) {
            block_residual(m[u], scale, v[u]);
            ss = block_squares(m[u], ss);
            if (p.dst.p != nullptr && there(u)) block_store<true>(p.dst.p + (int64_t)t * p.dst.nb, p.dst.type, first + u * step, p.H, m[u]);
        }
        if (!p.has_next) continue;
        const float inv = block_inverse_root(sum(block_pair_sum(ss), sums[turn + 1]), p.per, p.next_eps);
#pragma unroll
        for (int u = 0; u < kBlockUnits; ++u) {
            if (!there(u)) continue;
            block_scale(m[u], inv);
            block_scale(m[u], xw[u]);
            block_store<true>(p.next.p + (int64_t)t * p.next.nb, p.next.type, first + u * step, p.H, m[u]);
        }
    }
}

}  // namespace gx
