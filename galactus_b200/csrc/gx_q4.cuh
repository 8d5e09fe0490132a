// Products with 4-bit weights (Q4_0 and Q4_1, GGUF blocks read in place) and
// F16 / BF16 rows, for few rows per matrix (sm_100a):
//
//   Q4_0  y = sum over blocks  d * sum (q - 8) x
//   Q4_1  y = sum over blocks  (d * sum q x + m * sum x)
//
// plain (y_j = W_e x_j) or gated (act(G_e x_j, U_e x_j)).
//
// A job is 32 rows of a matrix (gated: 16 of each) against up to eight rows of x.
// A warp's step is 64 elements of K: codes become 16-bit floats without a rounding,
// the tensor cores (mma.sync m16n8k16) add their products with x in f32, and f32 fmas
// apply the block's d (and m). F16: q - 8, and for Q4_1 sum x from products with 1,
// which m + 8 d applies to; BF16: 16 + q, of which products with a constant take 24 or
// 16 times sum x off again. The roundings are those of f32 sums; the tensor cores
// cut where f32 would round (a step, for a half of one).
// (tcgen05 needs its matrices in shared memory, written and fenced: for a few rows
// that costs more than the products. With many, gx_gmm.cuh does just that.)
//
// Choices, as measured on a B200 (device time, calls in a row in a graph):
//   - x of the job's rows lies in shared memory, copied ahead by bulk copies: read
//     through L2 by each warp, 32 rows x 4096 x 14336 took 92 us, now 45.
//   - A ring per two warps that take the pairs of blocks in turn: TMA boxes of
//     32 rows x 8 pairs, or pieces of 16 bytes by cp.async where rows do not start on
//     16 bytes (2880 elements: 1620 bytes). Bulk copies, one a row, cost the issuing
//     warp 2800 cycles for 32 of them.
//   - Few jobs: warps share a job's K (p.share) and add their sums in their order, so
//     the same call gives the same bits.
// What bounds it: instructions and their latency. 264 MB of Q4_0 and one BF16 row: 76
// us, 3.5 TB/s (F16 67, 3.9; the copies by themselves 47). A step is some 180 of them
// and 86 cycles per SM, 2.2 a cycle of four that could be; no unit is full (the one for
// shifts, masks and permutations 51 %, tensor cores 28 %, DRAM 36 %). A warp issues
// every 5.6 cycles, four warps to a scheduler: 1.0 goes to the operation before, 0.9 to
// other warps' turns, 0.8 to full units, 0.7 to fetching instructions.
// 19 tokens x 8 of 64 experts, gated, 2048 x 1024, Q4_1: 46 us, 1.9 TB/s (two and three
// tiles of rows for the popular experts); one token, 8 of 128, 768 x 2048: 9.3 us, set-up
// and one round of jobs; 2880 x 2880, 4 experts, gated: 23 us, of which the copies of
// 16 bytes take 20.
#pragma once

#include <climits>

#include "gx_gmm.cuh"
#include "gx_q4_plan.h"

namespace gx {

struct Q4Params {
    CUtensorMap wmap, umap;   // their blocks as [words of a row, N, G], where rows lie on 16 bytes (boxes)
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
    int32_t warps;            // of a CTA
    int32_t share;            // warps that share a job's K (a divisor of the CTA's)
    int32_t cap;              // rows of x per tile
    int32_t buffers;          // tiles of x in shared memory
    int32_t boxes;
    int32_t lo, hi;           // rows of the groups that this launch is for
};

// ---------------------------------------------------------------- pieces

// (the first `bytes` of 16, zeros behind them)
__device__ __forceinline__ void q4_copy16(uint32_t dst, const uint8_t * src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t q4_lds(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

__device__ __forceinline__ uint2 q4_lds2(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}

// d = a x b + c
template <bool BF16>
__device__ __forceinline__ void q4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                       float c0, float c1, float c2, float c3) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// The codes of one word of a block (bytes 4t .. 4t+3: elements 4t + i in the
// low halves, 16 + 4t + i in the high ones) as pairs of 16-bit floats: (0, 1),
// (2, 3), (16, 17), (18, 19) from 4t on. A code goes into the mantissa of a
// power of two, all of it into the low byte: 16 + q (BF16) or 64 + q (F16), the
// high bytes are the same for all. (F16 codes as they stand, the subnormals
// q 2^-24, would take fewer operations, but the tensor cores add products of
// subnormals with ten bits less: 4e-5 of the result instead of 1e-7.)
// (F16: 72 comes off here, so that q - 8 enters the sums. With 64 + q in them and 72
// or 64 sum x taken off behind, what the tensor cores cut off was that of sums up to
// sixteen times the result: rows of mean 1, 1024 elements, 1.7e-6 of a Q4_0 result and
// 8.7e-7 of a Q4_1 one where f32 sums leave 1.8e-7. It rounds nothing, and a Q4_0
// step needs no product for sum x: 264 MB and one row 70 -> 67 us; Q4_1 keeps those
// products, 77 -> 81. BF16's 16 + q, and 24 or 16 sum x behind, stays at 1.1e-7 and
// 1.8e-7.)
// (Left shifts are products, which run beside the units for shifts, masks and
// byte permutations: those are what the kernel needs most.)
__device__ __forceinline__ uint32_t q4_times(uint32_t w, uint32_t by) {
    uint32_t v;
    asm("mul.lo.u32 %0, %1, %2;" : "=r"(v) : "r"(w), "r"(by));
    return v;
}
template <bool BF16>
__device__ __forceinline__ void q4_codes(uint32_t w, uint32_t (&a)[4]) {
    uint32_t lo, hi;
    if constexpr (BF16) {
        lo = (q4_times(w, 8u) & 0x78787878u) | 0x80808080u;
        hi = ((w >> 1) & 0x78787878u) | 0x80808080u;
    } else {
        lo = q4_times(w, 16u) & 0xF0F0F0F0u;
        hi = w & 0xF0F0F0F0u;
    }
    constexpr uint32_t top = BF16 ? 0x41414141u : 0x54545454u;
    a[0] = __byte_perm(lo, top, 0x4140);
    a[1] = __byte_perm(lo, top, 0x4342);
    a[2] = __byte_perm(hi, top, 0x4140);
    a[3] = __byte_perm(hi, top, 0x4342);
    if constexpr (!BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = q4_fma<false>(a[i], q4_one<false>(), 0xD480D480u);
    }
}
// The A operand of the products with x that are wanted beside the codes': BF16, what
// turns sums of 16 + q into those of q - 8 (Q4_0) or q (Q4_1), -24 or -16; F16, Q4_1:
// 1, for sum x itself
template <bool BF16, bool Q41>
__device__ __forceinline__ constexpr uint32_t q4_beside() {
    return BF16 ? (Q41 ? 0xC180C180u : 0xC1C0C1C0u) : 0x3C003C00u;
}

// the halves of a word, as f32
__device__ __forceinline__ float q4_low(uint32_t v) { return __low2float(*reinterpret_cast<const __half2 *>(&v)); }
__device__ __forceinline__ float q4_high(uint32_t v) { return __high2float(*reinterpret_cast<const __half2 *>(&v)); }

// ------------------------------------------------------------- the groups

// The groups of a launch. pre[i]: the tiles of rows before group i * per
struct Q4Groups {
    const int32_t * pre;
    int per, n;
    const int32_t * order;    // of the rows (global memory, or shared memory for ids), NULL: as they are
    const int32_t * expert;   // of group i (ids), NULL: i
    const int32_t * start;    // first row of group i (ids), NULL: offsets, or all rows
};

// A tile of a group's rows
struct Q4Tile {
    int group, before, tiles; // group, tiles of rows before it, and its own
    int e, row0, rows;        // expert, the tile's rows
};

// tile `at` of rows
__device__ __forceinline__ void q4_tile(const Q4Params & p, const Q4Groups & g, int at, Q4Tile & j) {
    const int i = tile_group(g.pre, (int)blockDim.x, at);
    j.group = i * g.per;
    j.before = g.pre[i];
    int lo, hi;
    for (;; ++j.group) {
        if (g.start != nullptr) {
            lo = g.start[j.group];
            hi = g.start[j.group + 1];
        } else {
            lo = p.offsets != nullptr ? p.offsets[j.group] : 0;
            hi = p.offsets != nullptr ? p.offsets[j.group + 1] : p.n_rows;
        }
        j.tiles = q4_group_tiles(lo, hi, p.n_rows, p.lo, p.hi, p.cap);
        if (at < j.before + j.tiles || j.group + 1 >= g.n) break;
        j.before += j.tiles;
    }
    j.e = g.start != nullptr ? g.expert[j.group] : j.group;
    // (a group's tiles are of one size, rather than full ones and a rest)
    const int size = (hi - lo - 1) / j.tiles + 1;
    j.row0 = lo + (at - j.before) * size;
    j.rows = min(size, hi - j.row0);
}

// As tile_prefix, for the groups that a thread looks at together: pre[i] is of
// group i * per, one per thread, and the last is the sum.
template <typename F>
__device__ __forceinline__ void q4_prefix(int32_t * pre, int32_t * wsum, int G, int per, int nt, int most, F && rows) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = blockDim.x;
    const int cap = most + 1;
    int sum = 0;
    for (int g = min(tid * per, G); g < min(tid * per + per, G); ++g) {
        const int2 r = rows(g);
        if (r.y > r.x) sum = min(sum + (r.y - r.x - 1) / nt + 1, cap);
    }
    int inc = sum;
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc = min(inc + v, cap);
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int before = inc - sum;
    for (int w = 0; w < warp; ++w) before += wsum[w];
    pre[tid] = before;
    if (tid == n - 1) {
        const bool over = before + sum > most;
        if (over) record_error(GX_DEVERR_DOMAIN);
        pre[n] = over ? 0 : before + sum;
    }
    __syncthreads();
}

// ------------------------------------------------------------- the kernel

// the warps that share a job
__device__ __forceinline__ void q4_sync(int team, int share) {
    if (share == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(32 * share) : "memory");
}

template <bool BF16, bool Q41, bool GLU>
__global__ void __launch_bounds__(32 * kQ4Warps, 1) k_q4(const __grid_constant__ Q4Params p) {
    constexpr int MT = kQ4Mt, CP = kQ4Pairs, S = kQ4Stages;
    constexpr int kPair = 2 * (Q41 ? 20 : 18);                      // bytes of 64 weights
    constexpr int kPitch = q4_pitch(Q41), kStage = q4_stage_bytes(Q41);
    constexpr int kRows = GLU ? 8 * MT : 16 * MT;                   // result rows of a job
    constexpr int kRed = kQ4Cols * kQ4Red;
    extern __shared__ __align__(128) uint8_t q4_smem_raw[];
    __shared__ int32_t wsum[kQ4Warps], pre[32 * kQ4Warps + 1];
    __shared__ int32_t s_order[kQ4MaxIds], s_key[kQ4MaxIds], s_lead[kQ4MaxIds], s_expert[kQ4MaxIds], s_start[kQ4MaxIds + 1];
    __shared__ uint64_t full[2], empty[2], ring_full[kQ4Warps / 2][S], ring_free[kQ4Warps / 2][S];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, W = p.warps;
    const int g = lane >> 2, t = lane & 3;
    float * red = reinterpret_cast<float *>(q4_smem_raw + W / 2 * S * kStage);
    uint8_t * xbuf = reinterpret_cast<uint8_t *>(red + W * kRed);
    const int x_pitch = (int)q4_x_pitch(p.K);

    griddep_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, (uint32_t)W);
        }
        for (int i = 0; i < W / 2 * S; ++i) {
            mbar_init(&ring_full[0][0] + i, p.boxes ? 1 : 64);
            mbar_init(&ring_free[0][0] + i, 2);
        }
        abort_flag = 0;
        mbar_fence_init();
    }
    griddep_wait();

    Q4Groups gr{pre, 1, p.G, p.order, nullptr, nullptr};
    if (p.ids != nullptr) {
        // rows by ascending expert, those of one expert in their order
        for (int r = tid; r < kQ4MaxIds; r += blockDim.x) {
            int key = r < p.n_rows ? p.ids[r] : -1;
            if (key >= p.G) {
                record_error(GX_DEVERR_DOMAIN);
                key = -1;
            }
            s_key[r] = key < 0 ? INT_MAX : key;
        }
        if (tid == 0) wsum[0] = wsum[1] = 0;
        __syncthreads();
        for (int r = tid; r < p.n_rows; r += blockDim.x) {
            const int key = s_key[r];
            int at = 0, same = 0;
            for (int i = 0; i < p.n_rows; ++i) {
                at += s_key[i] < key;
                same += s_key[i] == key && i < r;
            }
            s_lead[r] = same == 0 ? key : INT_MAX;                  // (the first row of each expert)
            s_order[at + same] = r;                                 // (rows of no expert come last)
            if (key == INT_MAX) continue;
            atomicAdd(&wsum[0], 1);
            if (same == 0) atomicAdd(&wsum[1], 1);
        }
        __syncthreads();
        for (int r = tid; r < p.n_rows; r += blockDim.x) {
            const int key = s_lead[r];
            if (key == INT_MAX) continue;
            int n = 0, at = 0;
            for (int i = 0; i < p.n_rows; ++i) {
                n += s_lead[i] < key;
                at += s_key[i] < key;
            }
            s_expert[n] = key;
            s_start[n] = at;
        }
        gr.n = wsum[1];
        if (tid == 0) s_start[gr.n] = wsum[0];
        __syncthreads();
        gr.order = s_order;
        gr.expert = s_expert;
        gr.start = s_start;
        gr.per = 1 + (gr.n - 1) / (int)blockDim.x;
        q4_prefix(pre, wsum, gr.n, gr.per, p.cap, p.most, [&](int i) { return make_int2(s_start[i], s_start[i + 1]); });
    } else if (p.offsets != nullptr) {
        gr.per = (p.G + (int)blockDim.x - 1) / (int)blockDim.x;
        q4_prefix(pre, wsum, p.G, gr.per, p.cap, p.most, [&](int i) {
            const int2 r = group_rows_of(p.offsets, i, p.n_rows);
            return r.y - r.x < p.lo || r.y - r.x > p.hi ? make_int2(0, 0) : r;
        });
    } else {
        q4_prefix(pre, wsum, 1, 1, p.cap, p.most, [&](int) { return make_int2(0, p.n_rows); });
    }

    // The CTA's run of jobs: tiles of rows, each with tiles of its matrix. Teams
    // of warps take the matrix tiles in turn, each warp a share of K.
    const int jobs = pre[blockDim.x] * p.rt;
    const int j0 = (int)((int64_t)jobs * blockIdx.x / gridDim.x), j1 = (int)((int64_t)jobs * (blockIdx.x + 1) / gridDim.x);
    if (j0 == j1) return;
    const int share = p.share, team = warp / share, member = warp - team * share, teams = W / share;
    const int pairs = p.K / 64;
    // A ring per two warps, which take its chunks' pairs of blocks in turn: a share
    // of K is theirs together. (Boxes start on 16 bytes: every fourth pair.)
    const int unit = p.boxes ? 4 : 1, parts = (pairs + unit - 1) / unit, of = share / 2, part2 = member >> 1, odd = member & 1;
    const int p0 = min(pairs, unit * (parts * part2 / of)), p1 = min(pairs, unit * (parts * (part2 + 1) / of));
    uint8_t * const ring_base = q4_smem_raw + (warp >> 1) * (S * kStage);
    const uint32_t ring = smem_u32(ring_base);
    uint64_t * const filled = ring_full[warp >> 1], * const freed = ring_free[warp >> 1];
    const int t0 = j0 / p.rt, t1 = (j1 - 1) / p.rt;                 // tiles of rows of the run
    auto m_begin = [&](int tile) { return tile == t0 ? j0 - t0 * p.rt : 0; };
    auto m_end = [&](int tile) { return tile == t1 ? j1 - t1 * p.rt : p.rt; };

    // ------------------------------------------------- the stream of chunks
    Q4Tile ahead;
    int ahead_tile = t0, ahead_m = m_begin(t0) + team, ahead_pair = p0, put = 0, issued = 0;
    auto ahead_enter = [&] {                                        // on to the team's next job
        while (ahead_tile <= t1 && ahead_m >= m_end(ahead_tile)) {
            ++ahead_tile;
            ahead_m = team;
            if (ahead_tile <= t1) q4_tile(p, gr, ahead_tile, ahead);
        }
    };
    q4_tile(p, gr, t0, ahead);
    Q4Tile job = ahead;
    ahead_enter();
    // Rows of a stage: 16 m + 8 h + g, or (gated) 16 h + 8 m + g: the gate's, the
    // up's. Where rows lie on 16 bytes they come as TMA boxes; elsewhere both warps
    // copy, eight lanes a row, pieces of 16 bytes from 16 bytes before its first one on.
    const int sub = lane >> 3, col = lane & 7;
    const int64_t up = p.w1 - p.w0;
    bool ok = true;
    auto issue = [&] {
        if ((odd && p.boxes) || ahead_tile > t1 || p0 >= p1) return;
        if (issued >= S) ok = ok && gmm_wait<1>(freed + put, (uint32_t)((issued / S - 1) & 1), &abort_flag);
        if (!ok) return;
        const int n = min(CP, p1 - ahead_pair);
        uint8_t * const stage = ring_base + put * kStage;
        if (p.boxes) {
            if (elect_one()) {
                mbar_arrive_expect_tx(filled + put, (uint32_t)kStage);
                tma_load_3d(stage, &p.wmap, ahead_pair * (kPair / 4), ahead_m * kRows, ahead.e, filled + put);
                if (GLU) tma_load_3d(stage + kStage / 2, &p.umap, ahead_pair * (kPair / 4), ahead_m * kRows, ahead.e, filled + put);
            }
            __syncwarp();
        } else {
            const int r0 = ahead_m * kRows + sub;
            const uint8_t * a = p.w0 + (int64_t)ahead.e * p.nb02 + (int64_t)r0 * p.nb01 + (int64_t)ahead_pair * kPair;
            const int skew = (int)(reinterpret_cast<uintptr_t>(a) & 15u), need = skew + n * kPair - col * 16;
            a += col * 16 - skew;
            const uint32_t to = smem_u32(stage) + (uint32_t)((16 * odd + sub) * kPitch + col * 16);
            const int half = GLU ? 0 : 16 * odd;                    // (each warp half of the stage's rows)
            if (GLU && odd) a += up;
#pragma unroll
            for (int i = 0; i < 4; ++i) {                           // row 4 i + sub of the half
                const int row = half + 4 * i;
                const uint8_t * from = a + (int64_t)row * p.nb01;
                if (r0 + row < p.N) {                               // (what lies in rows behind the last is not used)
#pragma unroll
                    for (int c = 0; c < (CP * kPair + 12 + 127) / 128; ++c)
                        if (c * 128 < need) q4_copy16(to + (uint32_t)(4 * i * kPitch + c * 128), from + c * 128, min(16, need - c * 128));
                }
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(filled + put)) : "memory");
        }
        put = put + 1 == S ? 0 : put + 1;
        ++issued;
        ahead_pair += n;
        if (ahead_pair >= p1) {
            ahead_pair = p0;
            ahead_m += teams;
            ahead_enter();
        }
    };
#pragma unroll
    for (int i = 0; i < S; ++i) issue();

    // ------------------------------------------------------ the tiles of x
    // Warp 0 copies the rows of tile i of the run, a lane a row.
    auto fetch = [&](const Q4Tile & j, int b) {
        if (lane == 0) mbar_arrive_expect_tx(full + b, (uint32_t)(j.rows * 2 * p.K));
        __syncwarp();
        if (lane < j.rows) {
            int row = j.row0 + lane;
            if (p.gather != 0) {
                const int o = gr.order[row];
                row = o / p.gather;
                if (o < 0 || row >= p.x_rows) row = 0;              // (its results are NaN)
            }
            bulk_g2s(xbuf + (b * p.cap + lane) * x_pitch, p.x + (int64_t)row * p.nb11, (uint32_t)(2 * p.K), full + b);
        }
    };
    int fetched = 1;
    if (warp == 0) fetch(job, 0);

    // ------------------------------------------------------------ the jobs
    int take = 0;
    uint32_t round = 0;
    const uint32_t beside = q4_beside<BF16, Q41>();
    for (int tile = t0; tile <= t1; ++tile) {
        const int i_tile = tile - t0, b = p.buffers == 2 ? i_tile & 1 : 0;
        Q4Tile next = job;
        if (tile < t1) q4_tile(p, gr, tile + 1, next);
        // the next tile of x, once its buffer is no longer read
        if (p.buffers == 2 && warp == 0 && tile < t1) {
            if (i_tile >= 1) ok = ok && gmm_wait<1>(empty + (b ^ 1), (uint32_t)(((i_tile - 1) >> 1) & 1), &abort_flag);
            if (ok) fetch(next, b ^ 1);
            fetched += ok;
        }
        // A wait that runs out makes what this warp adds to its team's sums NaN from here
        // on, and it hands nothing back: others then compute on what they have, and give up
        // behind it. Teams stay together.
        ok = gmm_wait<1>(full + b, (uint32_t)((p.buffers == 2 ? i_tile >> 1 : i_tile) & 1), &abort_flag) && ok;
        // (columns behind the last row repeat it)
        const uint32_t xs = smem_u32(xbuf) + (uint32_t)((b * p.cap + min(g, job.rows - 1)) * x_pitch + t * 8);
        for (int m = m_begin(tile) + team; m < m_end(tile); m += teams) {
            // where the lane's rows start inside their 16 bytes (rows 8 apart agree)
            const uint32_t low = (uint32_t)reinterpret_cast<uintptr_t>(p.w0) + (uint32_t)job.e * (uint32_t)p.nb02 +
                                 (uint32_t)(m * kRows + g) * (uint32_t)p.nb01;
            float acc[MT][2][2];                                   // [tile][half][column]
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][0][0] = acc[i][0][1] = acc[i][1][0] = acc[i][1][1] = 0.0f;

            for (int q0 = p0; q0 < p1; q0 += CP) {
                ok = gmm_wait<1>(filled + take, round, &abort_flag) && ok;
                const uint32_t at = ring + (uint32_t)(take * kStage + g * kPitch) + ((low + (uint32_t)(q0 * kPair)) & 15u);
                const int n_pairs = min(CP, p1 - q0);
#pragma unroll 2
                for (int q = odd; q < n_pairs; q += 2) {
                    // x: elements 4t .. and 16 + 4t .. of two blocks
                    uint2 x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = q4_lds2(xs + (uint32_t)((q0 + q) * 128 + i * 32));
                    // codes and scales of two blocks of the tile's rows
                    uint32_t a[MT][2][2][4];                        // [tile][block][half][pair of codes]
                    float d[MT][2][2], mn[MT][2][2];
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t r = at + (uint32_t)((GLU ? 16 * h + 8 * i : 16 * i + 8 * h) * kPitch) + (uint32_t)(q * kPair);
                            if constexpr (Q41) {
                                const uint32_t s0 = q4_lds(r), s1 = q4_lds(r + 20u);
                                q4_codes<BF16>(q4_lds(r + 4u + 4u * t), a[i][0][h]);
                                q4_codes<BF16>(q4_lds(r + 24u + 4u * t), a[i][1][h]);
                                d[i][0][h] = q4_low(s0);
                                d[i][1][h] = q4_low(s1);
                                // (BF16: sum x comes as -16 of it; F16: the codes' sums lack 8 d sum x)
                                mn[i][0][h] = BF16 ? __fmul_rn(-0.0625f, q4_high(s0)) : __fmaf_rn(8.0f, d[i][0][h], q4_high(s0));
                                mn[i][1][h] = BF16 ? __fmul_rn(-0.0625f, q4_high(s1)) : __fmaf_rn(8.0f, d[i][1][h], q4_high(s1));
                            } else {
                                const uint32_t s0 = q4_lds(r), s1 = q4_lds(r + 16u);
                                const uint32_t w0 = q4_lds(r + 4u * t), w1 = q4_lds(r + 4u + 4u * t);
                                q4_codes<BF16>(__byte_perm(w0, w1, 0x5432), a[i][0][h]);
                                q4_codes<BF16>(q4_lds(r + 20u + 4u * t), a[i][1][h]);
                                d[i][0][h] = q4_low(s0);
                                d[i][1][h] = q4_high(s1);
                            }
                        }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint2 lo = x[2 * k], hi = x[2 * k + 1];
                        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        if constexpr (BF16 || Q41) {
                            q4_mma<BF16>(s, beside, beside, beside, beside, lo.x, lo.y, 0.0f, 0.0f, 0.0f, 0.0f);
                            q4_mma<BF16>(s, beside, beside, beside, beside, hi.x, hi.y, s[0], s[1], s[2], s[3]);
                        }
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            float c[4];
                            q4_mma<BF16>(c, a[i][k][0][0], a[i][k][1][0], a[i][k][0][1], a[i][k][1][1], lo.x, lo.y, BF16 ? s[0] : 0.0f,
                                         BF16 ? s[1] : 0.0f, BF16 ? s[2] : 0.0f, BF16 ? s[3] : 0.0f);
                            q4_mma<BF16>(c, a[i][k][0][2], a[i][k][1][2], a[i][k][0][3], a[i][k][1][3], hi.x, hi.y, c[0], c[1], c[2], c[3]);
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int v = 0; v < 2; ++v) {
                                    acc[i][h][v] = __fmaf_rn(d[i][k][h], c[2 * h + v], acc[i][h][v]);
                                    if constexpr (Q41) acc[i][h][v] = __fmaf_rn(mn[i][k][h], s[v], acc[i][h][v]);
                                }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0 && ok) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(freed + take)) : "memory");
                if (++take == S) {
                    take = 0;
                    round ^= 1u;
                }
                issue();
            }

            // --------------------------- the warps' sums, added in their order
            float * part = red + team * share * kRed;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float * to = part + member * kRed + 2 * t * kQ4Red + 16 * i + 8 * h + g;
                    to[0] = ok ? acc[i][h][0] : kNan;
                    to[kQ4Red] = ok ? acc[i][h][1] : kNan;
                }
            q4_sync(team, share);
            for (int i = member * 32 + lane; i < kRows * job.rows; i += 32 * share) {
                const int c = i / kRows, r = i - c * kRows;         // (kRows is a power of two)
                const int row = m * kRows + r;
                if (row >= p.N) continue;
                const float * from = part + c * kQ4Red + (GLU ? (r >> 3) * 16 + (r & 7) : r);
                float v = from[0], u = GLU ? from[8] : 0.0f;
                for (int w = 1; w < share; ++w) {
                    v = __fadd_rn(v, from[w * kRed]);
                    if (GLU) u = __fadd_rn(u, from[w * kRed + 8]);
                }
                if (GLU) {
                    float gv[1] = {v}, uv[1] = {u};
                    gmm_act_all<1>(p, gv, uv);
                    v = gv[0];
                }
                const int j = job.row0 + c;
                bool nan = false;
                const int to = gmm_dst_row(p, j, gr.order != nullptr ? gr.order[j] : j, nan);
                if (nan && r == 0) record_error(GX_DEVERR_DOMAIN);
                if (to >= 0) store_out(p.dst + (int64_t)to * p.nbd1, row, nan ? kNan : v, p.out);
            }
            q4_sync(team, share);
        }
        // this warp is done with the tile of x
        __syncwarp();
        if (lane == 0 && ok) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(empty + b)) : "memory");
        if (p.buffers == 1 && warp == 0 && tile < t1) {
            ok = ok && gmm_wait<1>(empty + b, (uint32_t)(i_tile & 1), &abort_flag);
            if (ok) fetch(next, 0);
            fetched += ok;
        }
        job = next;
    }
    // copies in flight land before the CTA leaves
    if (!ok) asm volatile("cp.async.wait_all;" ::: "memory");
    volatile int none = 0;
    for (int i = 0; i < S && !ok; ++i)
        if (issued > i) gmm_wait<1>(filled + i, (uint32_t)((issued - 1 - i) / S & 1), &none);
    for (int i = max(0, fetched - p.buffers); i < fetched && !ok && warp == 0; ++i)
        gmm_wait<1>(full + (p.buffers == 2 ? i & 1 : 0), (uint32_t)((p.buffers == 2 ? i >> 1 : i) & 1), &none);
}

}  // namespace gx
