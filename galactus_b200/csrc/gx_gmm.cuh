// Products of ragged groups of rows with the F16 / BF16 matrices of their
// experts (sm_100a, tcgen05 + TMA).
//
//   plain  y_j = W_g x_j                      j in [offsets[g], offsets[g+1])
//   gated  y_j = act(G_g x_j, U_g x_j)
//
// The weights are the M side of the MMA (128 matrix rows, TMEM lanes) and the
// group's rows the N side (TMEM columns), so a group of c rows costs
// round_up(c, 16) columns and nothing is padded to a full tile: decode
// groups of one row and prefill groups of thousands run the same code.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gx_tc.cuh"

namespace gx {

constexpr int kGmmRows = 128;                  // matrix rows of a tile (MMA M)
constexpr int kGmmK = 64;                      // elements of K per stage: one 128-byte swizzled row
constexpr uint32_t kGmmATile = kGmmRows * 128u;
constexpr int kGmmMaxStages = 12;
constexpr int kGmmThreads = 192;               // producer, MMA issuer, 4 epilogue warps
constexpr int kGmmBox = 32;                    // rows of one TMA box of x (rows in place)

enum : int { GMM_F32 = 0, GMM_F16 = 1, GMM_BF16 = 2 };

struct GmmParams {
    CUtensorMap wmap;         // W (or G): [K, N, G], boxes 64 x 128
    CUtensorMap umap;         // U
    CUtensorMap xmap;         // x: [K, rows], boxes 64 x 32, or 64 x 1 for gathers
    const int32_t * offsets;  // [G + 1]
    const int32_t * order;    // [n_rows] or NULL
    int32_t G, n_rows, x_rows;
    int32_t N, K;
    int32_t gather;           // x row of j: order[j] / gather; 0: j itself
    int32_t scatter;          // y row of j: order[j] instead of j
    int32_t bf16;             // operand type
    int32_t out;              // GMM_*
    uint8_t * dst;
    int64_t nbd1;
    int32_t act;              // GX_ACT_*
    float alpha, limit;
    int32_t nt;               // rows of a group per tile (multiple of 16)
    int32_t stages;
    int32_t mt;               // tiles of 128 matrix rows
};

// ------------------------------------------------------------ PTX helpers

// D[tmem] (+)= A x B^T, f16 or bf16 operands, f32 accumulators, one thread
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum)
        : "memory");
}

// instruction descriptor of kind::f16: f32 accumulator, A and B of one type, both K-major
__host__ __device__ constexpr uint32_t umma_idesc_f16(bool bf16, uint32_t M, uint32_t N) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((N >> 3) << 17) | ((M >> 4) << 24);
}

__device__ __forceinline__ void tma_load_2d(void * dst, const CUtensorMap * map, int x, int y, uint64_t * bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}

// four rows of a one-row-box map (no multicast: this GPU's own memory)
__device__ __forceinline__ void tma_gather4(void * dst, const CUtensorMap * map, int x, int r0, int r1, int r2, int r3,
                                            uint64_t * bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5, %6}], [%7];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void gmm_arrive(uint64_t * bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// Bounded wait: gives up after two seconds, or once another role of the CTA has.
__device__ __forceinline__ bool gmm_wait(uint64_t * bar, uint32_t parity, volatile int * abort_flag) {
    if (mbar_test_wait(bar, parity)) return true;
    uint64_t t0 = 0;
    for (uint32_t i = 1;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63u) == 0u) {
            if (*abort_flag != 0) return false;
            const uint64_t t = global_ns();
            if (t0 == 0) t0 = t;
            else if (t - t0 > 2000000000ull) break;
        }
    }
    *abort_flag = 1;
    record_error(GX_DEVERR_TIMEOUT);
    return false;
}

#define kNan __int_as_float(0x7fc00000)

// rows [lo, hi) of group g, with borders that do not ascend or leave the rows
// reported and treated as empty groups
__device__ __forceinline__ int2 group_rows_of(const int32_t * offsets, int g, int n_rows) {
    const int lo = offsets[g], hi = offsets[g + 1];
    if (lo < 0 || hi < lo || hi > n_rows) {
        record_error(GX_DEVERR_DOMAIN);
        return make_int2(0, 0);
    }
    return make_int2(lo, hi);
}

// pre[g] = tiles of nt rows in the groups before g (G + 1 values), by the whole block
__device__ __forceinline__ void tile_prefix(int32_t * pre, int32_t * wsum, const int32_t * offsets, int G, int n_rows,
                                            int nt) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = blockDim.x;
    const int per = (G + n - 1) / n;
    const int g0 = min(tid * per, G), g1 = min(g0 + per, G);
    int sum = 0;
    for (int g = g0; g < g1; ++g) {
        const int2 r = group_rows_of(offsets, g, n_rows);
        pre[g] = sum;
        sum += (r.y - r.x + nt - 1) / nt;
    }
    int inc = sum;
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int before = inc - sum;
    for (int w = 0; w < warp; ++w) before += wsum[w];
    for (int g = g0; g < g1; ++g) pre[g] += before;
    if (tid == n - 1) pre[G] = before + sum;
    __syncthreads();
}

// group of row tile tt: the last g with pre[g] <= tt
__device__ __forceinline__ int tile_group(const int32_t * pre, int G, int tt) {
    int lo = 0, hi = G;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (pre[m] <= tt) lo = m; else hi = m;
    }
    return lo;
}

struct GmmTile {
    int g, m0, row0, cnt;
};

// tile t of the launch: the 128-row tiles of the matrix run fastest, so that
// CTAs at work together read the same rows and one expert's weights
__device__ __forceinline__ GmmTile gmm_tile(const GmmParams & p, const int32_t * pre, int t) {
    GmmTile r;
    const int tt = t / p.mt;
    r.m0 = (t - tt * p.mt) * kGmmRows;
    r.g = tile_group(pre, p.G, tt);
    const int lo = p.offsets[r.g], hi = p.offsets[r.g + 1];
    r.row0 = lo + (tt - pre[r.g]) * p.nt;
    r.cnt = min(p.nt, hi - r.row0);
    return r;
}

// x row of grouped row j (a bad index is reported; its result is not stored)
__device__ __forceinline__ int gmm_src_row(const GmmParams & p, int j) {
    if (p.gather == 0) return j;
    const int r = p.order[j] / p.gather;
    if (p.order[j] < 0 || r >= p.x_rows) {
        record_error(GX_DEVERR_DOMAIN);
        return 0;
    }
    return r;
}

// y row of grouped row j, -1 to skip it (no such row); nan: its x row does not exist
__device__ __forceinline__ int gmm_dst_row(const GmmParams & p, int j, bool & nan) {
    if (p.gather == 0 && p.scatter == 0) return j;
    const int o = p.order[j];
    nan = p.gather != 0 && (o < 0 || o / p.gather >= p.x_rows);
    if (p.scatter == 0) return j;
    if (o >= 0 && o < p.n_rows) return o;
    record_error(GX_DEVERR_DOMAIN);
    return -1;
}

__device__ __forceinline__ void store_out(uint8_t * row, int n, float v, int out) {
    if (out == GMM_F32) reinterpret_cast<float *>(row)[n] = v;
    else if (out == GMM_BF16) reinterpret_cast<__nv_bfloat16 *>(row)[n] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half *>(row)[n] = __float2half_rn(v);
}

__device__ __forceinline__ float gmm_act(const GmmParams & p, float g, float u) {
    return p.act == 0 ? act_swiglu(g, u) : act_swiglu_oai(g, u, p.alpha, p.limit);
}

__host__ __device__ constexpr uint32_t gmm_stage_bytes(bool glu, int nt) {
    return kGmmATile * (glu ? 2u : 1u) + (uint32_t)nt * 128u;
}

template <bool GLU>
__global__ void __launch_bounds__(kGmmThreads, 1) k_gmm(const __grid_constant__ GmmParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[kGmmMaxStages], empty[kGmmMaxStages], acc_full[2], acc_empty[2], drained;
    __shared__ uint32_t tslot;
    __shared__ int32_t wsum[kGmmThreads / 32];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint8_t * ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t stage_bytes = gmm_stage_bytes(GLU, p.nt);
    int32_t * pre = reinterpret_cast<int32_t *>(ring + (uint32_t)p.stages * stage_bytes);
    constexpr uint32_t kB = kGmmATile * (GLU ? 2u : 1u);   // the rows' tile inside a stage
    // TMEM columns: two accumulator buffers of (one or two) nt columns
    const uint32_t acc_cols = (uint32_t)p.nt * (GLU ? 2u : 1u);

    if (tid == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + i, 1);
            mbar_init(acc_empty + i, 4);
        }
        mbar_init(&drained, 1);
        abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(&tslot, 512);
        tmem_relinquish();
    }
    tile_prefix(pre, wsum, p.offsets, p.G, p.n_rows, p.nt);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = tslot;
    const int tiles = pre[p.G] * p.mt;
    const int nk = (p.K + kGmmK - 1) / kGmmK;

    if (warp == 0) {
        // ------------------------------------------------------- producer
        int c = 0, done = 0;           // chunks started; chunks whose stage was handed back
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            const GmmTile q = gmm_tile(p, pre, t);
            const int quads = (q.cnt + 3) >> 2;                  // rows in fours (the last repeats its final row)
            const int boxes = (q.cnt + kGmmBox - 1) / kGmmBox;
            const uint32_t bytes = kB + (p.gather ? (uint32_t)quads * 512u : (uint32_t)boxes * (kGmmBox * 128u));
            int r[2][4];
            if (p.gather) {
                for (int h = 0; h < 2; ++h)
                    for (int i = 0; i < 4; ++i) {
                        const int j = min((h * 32 + lane) * 4 + i, q.cnt - 1);
                        r[h][i] = gmm_src_row(p, q.row0 + j);
                    }
            }
            for (int kc = 0; kc < nk; ++kc, ++c) {
                const int s = c % p.stages;
                if (c >= p.stages) {
                    ok = __all_sync(0xffffffffu, gmm_wait(empty + s, (uint32_t)((c / p.stages - 1) & 1), &abort_flag));
                    if (!ok) break;
                    ++done;
                }
                uint8_t * st = ring + (uint32_t)s * stage_bytes;
                if (lane == 0) {
                    mbar_arrive_expect_tx(full + s, bytes);
                    tma_load_3d(st, &p.wmap, kc * kGmmK, q.m0, q.g, full + s);
                    if (GLU) tma_load_3d(st + kGmmATile, &p.umap, kc * kGmmK, q.m0, q.g, full + s);
                    if (!p.gather)
                        for (int b = 0; b < boxes; ++b)
                            tma_load_2d(st + kB + (uint32_t)b * (kGmmBox * 128u), &p.xmap, kc * kGmmK, q.row0 + b * kGmmBox,
                                        full + s);
                }
                __syncwarp();
                if (p.gather) {
                    if (lane < quads)
                        tma_gather4(st + kB + (uint32_t)lane * 512u, &p.xmap, kc * kGmmK, r[0][0], r[0][1], r[0][2], r[0][3],
                                    full + s);
                    if (lane + 32 < quads)
                        tma_gather4(st + kB + (uint32_t)(lane + 32) * 512u, &p.xmap, kc * kGmmK, r[1][0], r[1][1], r[1][2],
                                    r[1][3], full + s);
                }
            }
        }
        if (!ok) {
            // copies in flight land before the CTA leaves
            volatile int none = 0;
            for (int i = done; i < c; ++i) gmm_wait(full + i % p.stages, (uint32_t)((i / p.stages) & 1), &none);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------ MMA issuer
        int c = 0, it = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++it) {
            const GmmTile q = gmm_tile(p, pre, t);
            const uint32_t n = (uint32_t)((q.cnt + 15) & ~15);
            const uint32_t idesc = umma_idesc_f16(p.bf16 != 0, kGmmRows, n);
            const int b = it & 1;
            if (it >= 2) ok = __all_sync(0xffffffffu, gmm_wait(acc_empty + b, (uint32_t)((it / 2 - 1) & 1), &abort_flag));
            const uint32_t d = tbase + (uint32_t)b * acc_cols;
            for (int kc = 0; kc < nk && ok; ++kc, ++c) {
                const int s = c % p.stages;
                ok = __all_sync(0xffffffffu, gmm_wait(full + s, (uint32_t)((c / p.stages) & 1), &abort_flag));
                if (!ok) break;
                tc_fence_after();
                uint8_t * st = ring + (uint32_t)s * stage_bytes;
                if (lane == 0) {
                    const uint64_t da = umma_desc_sw128(st, 1024u), db = umma_desc_sw128(st + kB, 1024u);
                    const uint64_t du = umma_desc_sw128(st + kGmmATile, 1024u);
#pragma unroll
                    for (int i = 0; i < kGmmK / 16; ++i) {
                        mma_f16(d, da + (uint64_t)(2 * i), db + (uint64_t)(2 * i), idesc, kc | i);
                        if (GLU) mma_f16(d + p.nt, du + (uint64_t)(2 * i), db + (uint64_t)(2 * i), idesc, kc | i);
                    }
                    mma_commit(empty + s);
                    if (kc == nk - 1) mma_commit(acc_full + b);
                }
                __syncwarp();
            }
        }
        if (!ok) {
            volatile int none = 0;
            if (lane == 0) mma_commit(&drained);
            __syncwarp();
            gmm_wait(&drained, 0, &none);
        }
    } else {
        // -------------------------------------------------------- epilogue
        const int quad = warp & 3;             // TMEM lanes 32 * quad ..
        int it = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++it) {
            const GmmTile q = gmm_tile(p, pre, t);
            const int b = it & 1;
            ok = __all_sync(0xffffffffu, gmm_wait(acc_full + b, (uint32_t)((it / 2) & 1), &abort_flag));
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tbase + (uint32_t)b * acc_cols + ((uint32_t)quad << 21);
            const int n = q.m0 + quad * 32 + lane;
            for (int c0 = 0; c0 < q.cnt; c0 += 16) {
                uint32_t v[16], u[16];
                tmem_ld16(d + (uint32_t)c0, v);
                if (GLU) tmem_ld16(d + (uint32_t)(p.nt + c0), u);
                const int j = q.row0 + c0 + lane;
                bool nan = false;
                const int my = (lane < 16 && c0 + lane < q.cnt) ? gmm_dst_row(p, j, nan) : -1;
                const unsigned nans = __ballot_sync(0xffffffffu, nan);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int row = __shfl_sync(0xffffffffu, my, i);
                    if (row >= 0 && n < p.N) {
                        float a = __uint_as_float(v[i]);
                        if (GLU) a = gmm_act(p, a, __uint_as_float(u[i]));
                        store_out(p.dst + (int64_t)row * p.nbd1, n, (nans >> i) & 1u ? kNan : a, p.out);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) gmm_arrive(acc_empty + b);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tbase, 512);
    }
}

}  // namespace gx
