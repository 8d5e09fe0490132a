// Products with 4-bit weights (Q4_0 and Q4_1, GGUF blocks read in place) and
// F16 / BF16 rows, for few rows per matrix (sm_100a):
//
//   Q4_0  y = sum over blocks  d * sum (q - 8) x
//   Q4_1  y = sum over blocks  (d * sum q x + m * sum x)
//
// plain (y_j = W_e x_j) or gated (act(G_e x_j, U_e x_j)).
#pragma once

#include "gx_gmm.cuh"
#include "gx_q4_plan.h"

namespace gx {

struct Q4Params {
    const uint8_t * w0;       // W, or the gate matrices
    const uint8_t * w1;       // the up matrices
    int64_t nb01, nb02;
    const uint8_t * x;
    int64_t nb11;
    const int32_t * ids;      // [n_rows] expert of each row, or NULL
    const int32_t * offsets;  // [G + 1], or NULL
    const int32_t * order;    // [n_rows], or NULL
    int32_t G, n_rows, x_rows;
    int32_t N, K;
    int32_t gather, scatter;  // as GmmParams; with ids: gather >= 1, scatter = 1
    int32_t out;              // GMM_*
    uint8_t * dst;
    int64_t nbd1;
    int32_t act;
    float alpha, limit;
    int32_t rt;               // tiles of a matrix's rows
    int32_t most;             // tiles of rows that the groups can have
    int32_t entries;          // of the list of groups
};

// ---------------------------------------------------------------- pieces

__device__ __forceinline__ void q4_copy16(uint32_t dst, const uint8_t * src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void q4_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void q4_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t q4_lds(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

template <bool BF16>
__device__ __forceinline__ void q4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The codes of one word of a block (bytes 4t .. 4t+3: elements 4t + i in the
// low and 16 + 4t + i in the high halves) as pairs of 16-bit floats: (0, 2),
// (1, 3), (16, 18), (17, 19) from 4t on. A code is put into the upper bits of
// the mantissa of 16, which gives 16 + q. (F16 codes as they stand, the
// subnormals q 2^-24, would take one operation less, but the tensor cores add
// products of subnormals with ten bits less: 4e-5 of the result instead of 1e-7.)
template <bool BF16>
__device__ __forceinline__ void q4_codes(uint32_t w, uint32_t (&a)[4]) {
    if constexpr (BF16) {
        a[0] = ((w << 3) & 0x00780078u) | 0x41804180u;
        a[1] = ((w >> 5) & 0x00780078u) | 0x41804180u;
        a[2] = ((w >> 1) & 0x00780078u) | 0x41804180u;
        a[3] = ((w >> 9) & 0x00780078u) | 0x41804180u;
    } else {
        a[0] = ((w << 6) & 0x03C003C0u) | 0x4C004C00u;
        a[1] = ((w >> 2) & 0x03C003C0u) | 0x4C004C00u;
        a[2] = ((w << 2) & 0x03C003C0u) | 0x4C004C00u;
        a[3] = ((w >> 6) & 0x03C003C0u) | 0x4C004C00u;
    }
}
// What turns sums of the codes above into the wanted ones, as the A operand of
// a product with the same x: -24 (Q4_0: sums of q - 8) or -16 (Q4_1: of q)
template <bool BF16, bool Q41>
__device__ __forceinline__ constexpr uint32_t q4_shift() {
    return BF16 ? (Q41 ? 0xC180C180u : 0xC1C0C1C0u) : (Q41 ? 0xCC00CC00u : 0xCE00CE00u);
}

__device__ __forceinline__ float q4_half(uint32_t bits) {
    float f;
    asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.f32.f16 %0, h;\n\t}" : "=f"(f) : "r"(bits));
    return f;
}

// ------------------------------------------------------------- the groups

// The groups of a launch, in shared memory: pre[i], the tiles before group i.
struct Q4Groups {
    const int32_t * pre;
    const int32_t * order;    // of the rows (global memory, or shared memory for ids), NULL: as they are
    const int32_t * expert;   // of group i (ids), NULL: i
    const int32_t * start;    // first row of group i (ids), NULL: offsets, or all rows
    int n;
};

struct Q4Job {
    int group, m, tile;       // group, tile of the matrix's rows, tile of the group's rows
    int e, lo, hi, tiles;     // expert, the group's rows, tiles of them
};

__device__ __forceinline__ void q4_enter(const Q4Params & p, const Q4Groups & g, Q4Job & j) {
    j.tiles = g.pre[j.group + 1] - g.pre[j.group];
    if (g.start != nullptr) {
        j.e = g.expert[j.group];
        j.lo = g.start[j.group];
        j.hi = g.start[j.group + 1];
    } else {
        j.e = j.group;
        j.lo = p.offsets != nullptr ? p.offsets[j.group] : 0;
        j.hi = p.offsets != nullptr ? p.offsets[j.group + 1] : p.n_rows;
    }
}
__device__ __forceinline__ void q4_first(const Q4Params & p, const Q4Groups & g, int at, Q4Job & j) {
    // (the tiles of a group's rows run fastest, then the matrix's, then the groups)
    j.group = tile_group(g.pre, g.n, at / p.rt);
    const int tiles = g.pre[j.group + 1] - g.pre[j.group], in = at - g.pre[j.group] * p.rt;
    j.m = in / tiles;
    j.tile = in - j.m * tiles;
    q4_enter(p, g, j);
}
__device__ __forceinline__ void q4_next(const Q4Params & p, const Q4Groups & g, Q4Job & j) {
    if (++j.tile < j.tiles) return;
    j.tile = 0;
    if (++j.m < p.rt) return;
    j.m = 0;
    do ++j.group;
    while (j.group < g.n && g.pre[j.group + 1] == g.pre[j.group]);
    if (j.group < g.n) q4_enter(p, g, j);
}
// rows of a job: a group's tiles are of one size, rather than full ones and a rest
__device__ __forceinline__ int2 q4_rows(const Q4Job & j) {
    const int size = ((j.hi - j.lo - 1) / j.tiles + 8) / 8 * 8;
    const int lo = j.lo + j.tile * size;
    return make_int2(lo, min(size, j.hi - lo));
}

// ------------------------------------------------------------- the kernel

template <bool BF16, bool Q41, bool GLU, int NT>
__global__ void __launch_bounds__(kQ4Threads, 1) k_q4(const __grid_constant__ Q4Params p) {
    constexpr int MT = q4_mt(NT), CP = q4_pairs(NT), S = kQ4Stages;
    constexpr int kBlock = Q41 ? 20 : 18, kPair = 2 * kBlock;
    constexpr int kPitch = q4_pitch(Q41, NT), kStage = 16 * MT * kPitch;
    constexpr int kRows = GLU ? 8 * MT : 16 * MT;                   // result rows of a job
    constexpr int kRed = q4_red_pitch(NT);
    extern __shared__ __align__(128) uint8_t q4_smem_raw[];
    __shared__ int32_t wsum[kQ4Warps];
    __shared__ int32_t s_order[kQ4MaxIds], s_key[kQ4MaxIds], s_expert[kQ4MaxIds], s_start[kQ4MaxIds + 1];
    __shared__ int32_t s_groups;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    float * red = reinterpret_cast<float *>(q4_smem_raw + kQ4Warps * S * kStage);
    int32_t * pre = reinterpret_cast<int32_t *>(red + q4_buffers(NT) * kQ4Warps * 8 * NT * kRed);

    griddep_launch_dependents();
    griddep_wait();

    Q4Groups gr{pre, p.order, nullptr, nullptr, p.G};
    if (p.ids != nullptr) {
        // rows by ascending expert, those of one expert in their order
        int key = -1, at = 0, same = 0;
        if (tid < p.n_rows) {
            key = p.ids[tid];
            if (key >= p.G) {
                record_error(GX_DEVERR_DOMAIN);
                key = -1;
            }
        }
        if (tid < kQ4MaxIds) s_key[tid] = key;
        __syncthreads();
        if (key >= 0) {
            for (int i = 0; i < p.n_rows; ++i) {
                const int k = s_key[i];
                at += k >= 0 && k < key;
                same += k == key && i < tid;
            }
            s_order[at + same] = tid;
        }
        __syncthreads();
        if (same != 0) s_key[tid] = -1;           // only the first of each expert counts now
        const int rows = __syncthreads_count(key >= 0);
        const int groups = __syncthreads_count(key >= 0 && same == 0);
        if (key >= 0 && same == 0) {
            int i = 0;
            for (int k = 0; k < p.n_rows; ++k) i += s_key[k] >= 0 && s_key[k] < key;
            s_expert[i] = key;
            s_start[i] = at;
        }
        if (tid == 0) {
            s_start[groups] = rows;
            s_groups = groups;
        }
        __syncthreads();
        gr.n = s_groups;
        gr.order = s_order;
        gr.expert = s_expert;
        gr.start = s_start;
        tile_prefix(pre, wsum, gr.n, 8 * NT, p.most, [&](int i) { return make_int2(s_start[i], s_start[i + 1]); });
    } else if (p.offsets != nullptr) {
        tile_prefix(pre, wsum, p.G, 8 * NT, p.most, [&](int i) { return group_rows_of(p.offsets, i, p.n_rows); });
    } else {
        tile_prefix(pre, wsum, 1, 8 * NT, p.most, [&](int) { return make_int2(0, p.n_rows); });
    }
    const int jobs = pre[gr.n] * p.rt;
    const int j0 = (int)((int64_t)jobs * blockIdx.x / gridDim.x), j1 = (int)((int64_t)jobs * (blockIdx.x + 1) / gridDim.x);
    if (j0 == j1) return;

    // this warp's share of K, in pairs of blocks
    const int pairs = p.K / 64;
    const int p0 = (int)((int64_t)pairs * warp / kQ4Warps), p1 = (int)((int64_t)pairs * (warp + 1) / kQ4Warps);
    const uint32_t ring = smem_u32(q4_smem_raw) + (uint32_t)warp * (S * kStage);

    // ------------------------------------------------- the stream of chunks
    Q4Job ahead;
    q4_first(p, gr, j0, ahead);
    int ahead_job = j0, ahead_pair = p0, put = 0;
    const int sub = lane >> 3, col = lane & 7;
    auto issue = [&] {
        if (ahead_job < j1 && p0 < p1) {
            const int n = min(CP, p1 - ahead_pair), bytes = n * kPair;
            const uint32_t to = ring + (uint32_t)put * kStage;
            const int64_t base = (int64_t)ahead.e * p.nb02 + (int64_t)ahead_pair * kPair;
            const int r0 = ahead.m * kRows;
#pragma unroll
            for (int i = 0; i < 4 * MT; ++i) {
                const int s = 4 * i + sub;                         // row of the tile: 16 m + 8 h + g
                const int row = min(GLU ? r0 + (s >> 4) * 8 + (s & 7) : r0 + s, p.N - 1);
                const uint8_t * a = (GLU && ((s >> 3) & 1) ? p.w1 : p.w0) + base + (int64_t)row * p.nb01;
                const int skew = (int)(reinterpret_cast<uintptr_t>(a) & 15u), need = skew + bytes;
                const uint8_t * from = a - skew;
                const uint32_t at = to + (uint32_t)(s * kPitch);
#pragma unroll
                for (int c = 0; c < (CP * kPair + 12 + 127) / 128; ++c) {
                    const int off = (c * 8 + col) * 16;
                    if (off < need) q4_copy16(at + (uint32_t)off, from + off, min(16, need - off));
                }
            }
            put = put + 1 == S ? 0 : put + 1;
            ahead_pair += n;
            if (ahead_pair >= p1) {
                ahead_pair = p0;
                if (++ahead_job < j1) q4_next(p, gr, ahead);
            }
        }
        q4_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue();

    // ------------------------------------------------------------ the jobs
    Q4Job job;
    q4_first(p, gr, j0, job);
    int take = 0, last_group = -1, last_tile = -1;
    const uint8_t * xp[NT];
    const uint32_t shift = q4_shift<BF16, Q41>();
    for (int jb = j0; jb < j1; ++jb, q4_next(p, gr, job)) {
        const int2 rows = q4_rows(job);
        const int used = (rows.y + 7) / 8;                          // tiles of eight columns
        if (job.group != last_group || job.tile != last_tile) {
            last_group = job.group;
            last_tile = job.tile;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int j = rows.x + min(n * 8 + g, rows.y - 1);
                int row = j;
                if (p.gather != 0) {
                    const int o = gr.order[j];
                    row = o / p.gather;
                    if (o < 0 || row >= p.x_rows) row = 0;          // (its result is NaN)
                }
                xp[n] = p.x + (int64_t)row * p.nb11 + t * 8;
            }
        }
        // where the rows of the tile start inside their 16 bytes
        uint32_t low[MT][2];
        {
            const uint32_t e = (uint32_t)job.e * (uint32_t)p.nb02;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = min(job.m * kRows + (GLU ? 8 * m + g : 16 * m + 8 * h + g), p.N - 1);
                    low[m][h] = (uint32_t)reinterpret_cast<uintptr_t>(GLU && h ? p.w1 : p.w0) + e + (uint32_t)row * (uint32_t)p.nb01;
                }
        }
        uint64_t acc[MT][NT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[m][n][0] = acc[m][n][1] = 0ull;

        for (int q0 = p0; q0 < p1; q0 += CP) {
            issue();
            q4_wait<S - 1>();
            __syncwarp();
            const uint32_t st = ring + (uint32_t)take * kStage;
            uint32_t at[MT][2];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    at[m][h] = st + (uint32_t)((16 * m + 8 * h + g) * kPitch) + ((low[m][h] + (uint32_t)(q0 * kPair)) & 15u);
            const int n_pairs = min(CP, p1 - q0);
#pragma unroll 2
            for (int q = 0; q < n_pairs; ++q) {
                // codes and scales of two blocks of the tile's rows
                uint32_t a[MT][2][2][4];                            // [tile][block][half][pair of codes]
                float d[MT][2][2], mn[MT][2][2];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t b = at[m][h] + (uint32_t)(q * kPair);
                        if constexpr (Q41) {
                            const uint32_t s0 = q4_lds(b), s1 = q4_lds(b + 20u);
                            q4_codes<BF16>(q4_lds(b + 4u + 4u * t), a[m][0][h]);
                            q4_codes<BF16>(q4_lds(b + 24u + 4u * t), a[m][1][h]);
                            d[m][0][h] = q4_half(s0 & 0xFFFFu);
                            mn[m][0][h] = q4_half(s0 >> 16);
                            d[m][1][h] = q4_half(s1 & 0xFFFFu);
                            mn[m][1][h] = q4_half(s1 >> 16);
                            mn[m][0][h] *= -0.0625f;                // (sum x comes as -16 sum x)
                            mn[m][1][h] *= -0.0625f;
                        } else {
                            const uint32_t s0 = q4_lds(b), s1 = q4_lds(b + 16u);
                            const uint32_t w0 = q4_lds(b + 4u * t), w1 = q4_lds(b + 4u + 4u * t);
                            q4_codes<BF16>(__byte_perm(w0, w1, 0x5432), a[m][0][h]);
                            q4_codes<BF16>(q4_lds(b + 20u + 4u * t), a[m][1][h]);
                            d[m][0][h] = q4_half(s0 & 0xFFFFu);
                            d[m][1][h] = q4_half(s1 >> 16);
                        }
                    }
                const int64_t xo = (int64_t)(q0 + q) * 128;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (NT > 1 && n >= used) break;
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint2 lo = __ldg(reinterpret_cast<const uint2 *>(xp[n] + xo + b * 64));
                        const uint2 hi = __ldg(reinterpret_cast<const uint2 *>(xp[n] + xo + b * 64 + 32));
                        const uint32_t l0 = __byte_perm(lo.x, lo.y, 0x5410), l1 = __byte_perm(lo.x, lo.y, 0x7632);
                        const uint32_t h0 = __byte_perm(hi.x, hi.y, 0x5410), h1 = __byte_perm(hi.x, hi.y, 0x7632);
                        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        q4_mma<BF16>(s, shift, shift, shift, shift, l0, l1);
                        q4_mma<BF16>(s, shift, shift, shift, shift, h0, h1);
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            float c[4] = {s[0], s[1], s[2], s[3]};
                            q4_mma<BF16>(c, a[m][b][0][0], a[m][b][1][0], a[m][b][0][1], a[m][b][1][1], l0, l1);
                            q4_mma<BF16>(c, a[m][b][0][2], a[m][b][1][2], a[m][b][0][3], a[m][b][1][3], h0, h1);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                acc[m][n][h] = fma_x2(f2pack(d[m][b][h], d[m][b][h]), f2pack(c[2 * h], c[2 * h + 1]), acc[m][n][h]);
                                if constexpr (Q41)
                                    acc[m][n][h] = fma_x2(f2pack(mn[m][b][h], mn[m][b][h]), f2pack(s[0], s[1]), acc[m][n][h]);
                            }
                        }
                    }
                }
            }
            take = take + 1 == S ? 0 : take + 1;
            __syncwarp();
        }

        // ------------------------------- the warps' sums, added in their order
        float * part = red + (q4_buffers(NT) == 2 ? jb & 1 : 0) * (kQ4Warps * 8 * NT * kRed);
        float * mine = part + warp * (8 * NT * kRed);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (NT > 1 && n >= used) break;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v0, v1;
                    f2unpack(acc[m][n][h], v0, v1);
                    float * to = mine + (n * 8 + 2 * t) * kRed + 16 * m + 8 * h + g;
                    to[0] = v0;
                    to[kRed] = v1;
                }
            }
        __syncthreads();
        for (int i = tid; i < kRows * rows.y; i += kQ4Threads) {
            const int c = i / kRows, r = i - c * kRows;             // (kRows is a power of two)
            const int row = job.m * kRows + r;
            if (row >= p.N) continue;
            const float * from = part + c * kRed + (GLU ? (r >> 3) * 16 + (r & 7) : r);
            float v = 0.0f, u = 0.0f;
#pragma unroll
            for (int w = 0; w < kQ4Warps; ++w) {
                v = __fadd_rn(v, from[w * (8 * NT * kRed)]);
                if (GLU) u = __fadd_rn(u, from[w * (8 * NT * kRed) + 8]);
            }
            if (GLU) {
                float gv[1] = {v}, uv[1] = {u};
                gmm_act_all<1>(p, gv, uv);
                v = gv[0];
            }
            const int j = rows.x + c;
            bool nan = false;
            const int to = gmm_dst_row(p, j, gr.order != nullptr ? gr.order[j] : j, nan);
            if (nan && r == 0) record_error(GX_DEVERR_DOMAIN);
            if (to >= 0) store_out(p.dst + (int64_t)to * p.nbd1, row, nan ? kNan : v, p.out);
        }
        if (q4_buffers(NT) == 1) __syncthreads();
    }
}

}  // namespace gx
