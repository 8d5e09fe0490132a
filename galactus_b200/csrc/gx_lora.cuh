// Low-rank deltas of many requests' adapters beside a projection they share
// (sm_100a, tcgen05 + TMA):
//
//   y_j = base_j + B_g (s_g A_g x_j)          j in the rows of group g
//
// A_g [rank, K] and B_g [N, rank] are F16 or BF16, x of the same type, base
// and y F32, F16 or BF16.
//
// ONE kernel does both products: a cluster of C CTAs takes up to 32 rows of a
// group. Each CTA multiplies its share of K (A_g on the M side, the rows on
// the N side), the partial h of the CTAs meet in shared memory over the
// cluster and are summed in CTA order, and each CTA then forms its share of
// the N results, adds base and writes them. h never leaves the SMs, and a
// call with one row still uses eight SMs.
//
// h is held in 32 bits. For the second product it is split into parts of the
// operand type that sum to it (three BF16 parts: 24 bits; two F16 parts: 22
// bits below the row's largest value, the row scaled by a power of two first
// so that no h overflows F16), all multiplied with the same B tile in shared
// memory: the deltas keep f32 accuracy for two extra MMAs per 16 ranks, which
// the memory-bound kernel has time for. The tensor cores' accumulators truncate
// (for sums of one sign 4.8e-5 of the sum at K = 7168, 1.6e-4 at 28672), so
// for f32 results each takes 512 elements of K and the sums of the accumulators
// are rounded adds (3.1e-6 and 1.4e-6 then; 8192 routed rows take 41 us with
// it, 40 without). Six accumulators let a tile of K = 2048 be multiplied
// while the one before it is finished (1.3 us more with two).
//
// Ranks differ by adapter: rows of A and columns of B behind an adapter's
// rank may hold anything and do not reach the result.
//
// Bounded by latency. On a B200 (calls in a row on one set of inputs; in
// brackets on changing ones, called from Python) a call of one row takes 12 us
// [14], of which 2 are the launch's set-up, 1.5 the first product, 2.5 the
// exchange and 2 the second; 64 requests on 48 adapters of ranks 8 to 64
// (K = N = 4096, 15 MB) 22 us [25] in clusters of four; 8192 routed rows in 250
// groups (rank 16, K 2048, N 768, f32, 64 MB) 41 us [47 to 55]. There a CTA has
// about two tiles; at gather4's rate (four rows of 128 bytes in 24 cycles) the
// copies of x account for a third of the time, and the rest is not broken down.
// What helped: rows that follow one another are copied as one box, two CTAs
// share an SM where the ranks allow, base is fetched into L2 at the start of a
// tile and into registers a result tile ahead (52 us without, at the time), and
// the results of a tile are issued between the chunks of the next one (52 us to
// 46). Tiles of 64 rows took 87 us: fewer fit on an SM, and routed groups are
// shorter.
#pragma once

#include "gx_gmm.cuh"

namespace gx {

struct LoraParams {
    CUtensorMap amap;         // A: [K, rank, G], boxes 64 x ra
    CUtensorMap bmap;         // B: [rank, N, G], boxes min(ra, 64) x 128
    CUtensorMap xmap;         // x: [K, rows], boxes 64 x 1, gathered
    CUtensorMap rmap;         // x: boxes 64 x 32
    const int32_t * offsets;  // [G + 1]
    const int32_t * order;    // [n_rows] or NULL: rows in place
    const int32_t * ranks;    // [G / n_as] or NULL: all `rank`
    const float * scale;      // [G / n_as] or NULL: 1
    const uint8_t * base;
    uint8_t * dst;
    int64_t nbb, nbd;
    int32_t G, n_as, n_rows, x_rows, gather;
    int32_t N, K, rank;
    int32_t ra;               // rank rounded up to 16, 32, 64 or 128
    int32_t bf16, out;
    int32_t copy;             // base is not dst: rows without an adapter are copied
    int32_t stages;
    int32_t most;             // tiles that the rows can have, those without an adapter among them
    int32_t seg;              // chunks that one accumulator of h sums (0: all)
};

// byte of 16-byte piece c of row r in such a block: the piece's number is
// XOR-ed with the address bits from 7 up
__device__ __forceinline__ uint32_t lora_swizzle(uint32_t row_bytes, int r, int c) {
    const uint32_t off = (uint32_t)r * row_bytes + (uint32_t)c * 16u;
    return off ^ (((off >> 7) & (row_bytes / 16u - 1u)) << 4);
}
// shared-memory descriptor of such a block, K-major (layout types 2, 4, 6: 128-, 64- and 32-byte swizzle)
__device__ __forceinline__ uint64_t lora_desc(const void * smem, uint32_t row_bytes) {
    const uint64_t layout = row_bytes == 128u ? 2u : row_bytes == 64u ? 4u : 6u;
    return (uint64_t)((smem_u32(smem) >> 4) & 0x3FFFu) | ((uint64_t)1u << 16) | ((uint64_t)((row_bytes * 8u) >> 4) << 32) |
           (1ull << 46) | (layout << 61);
}

__device__ __forceinline__ float4 ld_peer4(const float * p, int cta) {
    float4 v;
    asm volatile(
        "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %4, %5;\n\t"
        "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [r];\n\t}"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
        : "r"(smem_u32(p)), "r"(cta)
        : "memory");
    return v;
}

struct LoraTile {
    int g, row0, cnt;
    int rank;         // 0: the rows have no adapter
};

__device__ __forceinline__ int2 lora_rows(const LoraParams & p, int g) {
    if (g < p.G) return group_rows_of(p.offsets, g, p.n_rows);
    const int lo = p.offsets[p.G];
    if (lo < 0 || lo > p.n_rows || p.offsets[0] != 0) {
        record_error(GX_DEVERR_DOMAIN);
        return make_int2(0, 0);
    }
    return p.copy ? make_int2(lo, p.n_rows) : make_int2(0, 0);
}

__device__ __forceinline__ LoraTile lora_tile(const LoraParams & p, const int32_t * pre, int t) {
    LoraTile q;
    q.g = tile_group(pre, p.G + 1, t);
    const int lo = p.offsets[q.g], hi = q.g < p.G ? p.offsets[q.g + 1] : p.n_rows;
    q.row0 = lo + (t - pre[q.g]) * kLoraRows;
    q.cnt = min(kLoraRows, hi - q.row0);
    q.rank = 0;
    if (q.g < p.G) {
        q.rank = p.ranks != nullptr ? p.ranks[q.g / p.n_as] : p.rank;
        if (q.rank < 0 || q.rank > p.rank) {
            record_error(GX_DEVERR_DOMAIN);
            q.rank = 0;
        }
    }
    return q;
}

// y row of grouped row j (-1: none), and whether its x row exists
__device__ __forceinline__ int lora_row(const LoraParams & p, int j, bool & bad_x) {
    const int row = p.order != nullptr ? p.order[j] : j;
    bad_x = row < 0 || row / p.gather >= p.x_rows;
    if (row >= 0 && row < p.n_rows) return row;
    record_error(GX_DEVERR_DOMAIN);
    return -1;
}

__device__ const uint4 g_no_piece = {0u, 0u, 0u, 0u};

// The base of a warp's 32 x 32 tile of results, loaded ahead of the deltas:
// lane's 16-byte pieces, rows of the 32 columns by `my` (lane i: column i).
template <typename T>
struct LoraBase {
    static constexpr int kPer = 16 / (int)sizeof(T), kLanes = 32 / kPer, kCols = 32 / kLanes, kPieces = 32 / kCols;
    uint4 old[kPieces];
    __device__ __forceinline__ void load(const LoraParams & p, int my, int n0, bool vec) {
        const int lane = threadIdx.x & 31, n = n0 + lane % kLanes * kPer;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int row = __shfl_sync(0xffffffffu, my, i * kCols + lane / kLanes);
            // (always a load: one under a condition is waited for where its branches meet)
            const bool have = vec && n + kPer <= p.N && row >= 0;
            old[i] = *reinterpret_cast<const uint4 *>(have ? p.base + (int64_t)row * p.nbb + (int64_t)n * (int)sizeof(T)
                                                           : reinterpret_cast<const uint8_t *>(&g_no_piece));
        }
    }
    // plus 16 staged columns of f32 deltas ([column][32 rows of B], columns 16 * half ..), rounded, to the result rows
    __device__ __forceinline__ void add(const LoraParams & p, const float * stage, int half, int my, int n0, bool vec) {
        const int lane = threadIdx.x & 31, sub = lane % kLanes, n = n0 + sub * kPer;
#pragma unroll
        for (int i = 0; i < kPieces / 2; ++i) {
            const int col = i * kCols + lane / kLanes;
            const int row = __shfl_sync(0xffffffffu, my, 16 * half + col);
            if (row < 0) continue;
            float d[kPer];
#pragma unroll
            for (int e = 0; e < kPer; e += 4)
                *reinterpret_cast<float4 *>(d + e) = *reinterpret_cast<const float4 *>(stage + col * 32 + sub * kPer + e);
            T * out = reinterpret_cast<T *>(p.dst + (int64_t)row * p.nbd) + n;
            if (vec && n + kPer <= p.N) {
                uint4 v = half ? old[kPieces / 2 + i] : old[i];
                T * t = reinterpret_cast<T *>(&v);
#pragma unroll
                for (int e = 0; e < kPer; ++e) t[e] = round_to<T>((float)t[e] + d[e]);
                *reinterpret_cast<uint4 *>(out) = v;
            } else {
                const T * was = reinterpret_cast<const T *>(p.base + (int64_t)row * p.nbb) + n;
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    if (n + e < p.N) out[e] = round_to<T>((float)was[e] + d[e]);
            }
        }
    }
};

template <typename T>
__device__ __forceinline__ void lora_copy_row(const LoraParams & p, int row, int first, int step) {
    const T * s = reinterpret_cast<const T *>(p.base + (int64_t)row * p.nbb);
    T * d = reinterpret_cast<T *>(p.dst + (int64_t)row * p.nbd);
    const bool vec = ((reinterpret_cast<uintptr_t>(s) | reinterpret_cast<uintptr_t>(d)) & 15u) == 0;
    constexpr int kPer = 16 / (int)sizeof(T);
    const int pieces = vec ? p.N / kPer : 0;
    for (int i = first; i < pieces; i += step) reinterpret_cast<uint4 *>(d)[i] = reinterpret_cast<const uint4 *>(s)[i];
    for (int i = pieces * kPer + first; i < p.N; i += step) d[i] = s[i];
}

// eight values of h as vectors of the operand type that sum to them: three of
// BF16 (24 bits), two of F16 (22)
template <typename T>
__device__ __forceinline__ void split_part(float (&rest)[8], uint4 & out) {
    T * v = reinterpret_cast<T *>(&out);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = round_to<T>(rest[i]);
        const float d = __fsub_rn(rest[i], (float)v[i]);
        rest[i] = fabsf(d) < __int_as_float(0x7f800000) ? d : 0.0f;          // (an infinity or NaN stays in the first part)
    }
}
__host__ __device__ constexpr int lora_parts(bool bf16) { return bf16 ? 3 : 2; }

__global__ void __launch_bounds__(kLoraThreads, 2) k_lora(const __grid_constant__ LoraParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[kLoraMaxStages], empty[kLoraMaxStages], b_full[2], b_empty[2], b_fixed[2], d2_full[2], d2_empty[2];
    __shared__ uint64_t d1_full[kLoraSums], d1_empty[kLoraSums], part_full, part_free, h_full, h_empty, drained;
    __shared__ int4 gather_mem[2 * kLoraRows / 4];
    __shared__ uint32_t tslot;
    __shared__ int32_t wsum[kLoraThreads / 32];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t ctas, rank_of;
    asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(ctas));
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(rank_of));
    const int C = (int)ctas, me = (int)rank_of;
    const int unit = (int)blockIdx.x / C, units = (int)gridDim.x / C;
    const uint32_t blocks = lora_blocks(p.ra), stage_bytes = lora_stage_bytes(p.ra), b_block = lora_b_block(p.ra);
    const uint32_t b_bytes = blocks * b_block, h_block = lora_h_block(p.ra), row_bytes = lora_row(p.ra);
    // the ring comes first: an MMA over 128 rows of A reads past the last
    // stage's rows into what follows (16 KB at most; lanes that nobody looks at)
    uint8_t * ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t * bring = ring + (uint32_t)p.stages * stage_bytes;
    uint8_t * hbuf = bring + 2u * b_bytes;
    float * part = reinterpret_cast<float *>(hbuf + 3u * blocks * h_block);    // [row][ra]
    float * staging = part + kLoraRows * p.ra;
    float * esc = staging + kLoraStaging / 4;                                  // [row] power of two of its h
    int32_t * pre = reinterpret_cast<int32_t *>(esc + kLoraRows);

    if (tid == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(b_full + i, 1);
            mbar_init(b_empty + i, 1);
            mbar_init(b_fixed + i, 1);
            mbar_init(d2_full + i, 1);
            mbar_init(d2_empty + i, kLoraEpiWarps);
        }
        for (int i = 0; i < kLoraSums; ++i) {
            mbar_init(d1_full + i, 1);
            mbar_init(d1_empty + i, kLoraEpiWarps);
        }
        mbar_init(&part_full, (uint32_t)(kLoraEpiWarps * C));
        mbar_init(&part_free, (uint32_t)(kLoraEpiWarps * C));
        mbar_init(&h_full, kLoraEpiWarps);
        mbar_init(&h_empty, 1);
        mbar_init(&drained, 1);
        abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) gmm_tmem_alloc<1>(&tslot, kLoraTmem);
    tile_prefix(pre, wsum, p.G + 1, kLoraRows, p.most, [&](int g) { return lora_rows(p, g); });
    tc_fence_before();
    if (C > 1) cluster_sync_all(); else __syncthreads();
    tc_fence_after();
    const uint32_t tbase = tslot;
    const uint32_t d1 = tbase, d2 = tbase + (uint32_t)(kLoraSums * kLoraRows);
    const int tiles = pre[p.G + 1];
    const int nk = (p.K + kLoraK - 1) / kLoraK;
    const int k0 = nk * me / C, k1 = nk * (me + 1) / C;                        // this CTA's chunks of K
    const int nn = (p.N + 127) / 128, n_lo = nn * me / C, n_hi = nn * (me + 1) / C;        // this CTA's result tiles
    const int nseg = p.seg && k1 > k0 ? (k1 - k0 + p.seg - 1) / p.seg : 1;                 // sums of h per tile

    if (warp == 0 || warp == 2) {
        // ------ A by TMA tiles and the rows of x by tile::gather4: two warps,
        // chunk by chunk in turn (one thread's issue rate would set the pace;
        // the stage count is even, so a stage stays with one of them)
        const int gw = warp >> 1;
        int32_t * rows = reinterpret_cast<int32_t *>(gather_mem + gw * 8);
        int c0 = 0;                    // chunks of the CTA so far
        RingPos at;
        bool ok = true;
        for (int t = unit; t < tiles && ok; t += units) {
            const LoraTile q = lora_tile(p, pre, t);
            if (q.rank == 0) continue;
            const int quads = (q.cnt + 3) >> 2;                          // rows in fours; those behind the last repeat it
            bool bad = false;
            const int row = lora_row(p, q.row0 + min(lane, q.cnt - 1), bad);
            if (bad) record_error(GX_DEVERR_DOMAIN);
            const int from = bad || row < 0 ? 0 : row / p.gather;
            __syncwarp();
            rows[lane] = from;
            __syncwarp();
            // rows that follow one another (a request's chunk of a prefill) are one box
            const int first = __shfl_sync(0xffffffffu, from, 0);
            const bool run = __all_sync(0xffffffffu, lane >= q.cnt || from == first + lane) && q.cnt > 4;
            const uint32_t bytes = 2u * ((uint32_t)p.ra * 128u + (run ? kLoraXTile : (uint32_t)quads * 512u));
            if (elect_one()) {
                int4 of[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) of[i] = *reinterpret_cast<const int4 *>(rows + i * 4);
                RingPos on = at;
                int c = c0;
                for (int kc = k0; kc < k1; ++kc, ++c, on.next(p.stages)) {
                    if ((c & 1) != gw) continue;
                    if (on.round != 0) {
                        ok = gmm_wait_one<1>(empty + on.s, (on.round - 1u) & 1u, &abort_flag);
                        if (!ok) break;
                    }
                    uint8_t * st = ring + (uint32_t)on.s * stage_bytes;
                    mbar_arrive_expect_tx(full + on.s, bytes);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        // (past the end of K, TMA fills in zeros)
                        const int x = kc * kLoraK + half * kGmmK;
                        tma_load_3d(st + 2u * kLoraXTile + (uint32_t)half * (uint32_t)p.ra * 128u, &p.amap, x, 0, q.g, full + on.s);
                        uint8_t * xt = st + (uint32_t)half * kLoraXTile;
                        if (run) gmm_tma_2d<1>(xt, &p.rmap, x, first, full + on.s);
                        else {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                if (i < quads) gmm_gather4<1>(xt + i * 512, &p.xmap, x, of[i].x, of[i].y, of[i].z, of[i].w, full + on.s);
                        }
                    }
                }
                if (!ok) {
                    // copies in flight land before the CTA leaves
                    volatile int none = 0;
                    for (int i = max(0, c - p.stages); i < c; ++i)
                        if ((i & 1) == gw) gmm_wait_one<1>(full + i % p.stages, (uint32_t)((i / p.stages) & 1), &none);
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            c0 += k1 - k0;
            at.skip(k1 - k0, p.stages);
        }
        // (the issuer's last commits arrive before the CTA leaves: those of the
        // ring are waited for here, those of B and h by the roles that use them)
        bool last = ok;
        for (int i = max(0, c0 - p.stages); i < c0 && last; ++i)
            if ((i & 1) == gw) last = gmm_wait<1>(empty + i % p.stages, (uint32_t)((i / p.stages) & 1), &abort_flag);
        if (ok && !last) {
            volatile int none = 0;
            for (int i = max(0, c0 - p.stages); i < c0; ++i)
                if ((i & 1) == gw) gmm_wait<1>(full + i % p.stages, (uint32_t)((i / p.stages) & 1), &none);
        }
    } else if (warp == 1) {
        // ----------------------------------------------------- MMA issuer
        if (elect_one()) {
            int it = 0, bc = 0;
            RingPos at;
            bool ok = true;
            const uint64_t a0 = umma_desc_sw128(ring + 2u * kLoraXTile, 1024u), x0 = umma_desc_sw128(ring, 1024u);
            const uint64_t b0 = lora_desc(bring, row_bytes), h0 = lora_desc(hbuf, row_bytes);
            const int parts = lora_parts(p.bf16 != 0);
            // The results of a tile are issued between the chunks of the next
            // tile's h, as its own h and the tiles of B become ready: neither
            // the exchange over the cluster nor the copies of x hold the other up.
            LoraTile last{};
            int next = 0;                              // result tile of `last` to issue
            bool open = false, have_h = false;
            auto ready = [&](uint64_t * bar, uint32_t parity, bool wait) {
                if (!wait) return mbar_test_wait(bar, parity);
                ok = ok && gmm_wait_one<1>(bar, parity, &abort_flag);
                return ok;
            };
            auto results = [&](bool wait) {            // (j of `last`: it - 1)
                const uint32_t idesc = umma_idesc_f16(p.bf16 != 0, 128, (uint32_t)((last.cnt + 15) & ~15));
                if (!have_h) have_h = ready(&h_full, (uint32_t)((it - 1) & 1), wait);
                if (!have_h) return;
                const int steps = (last.rank + 15) / 16;
                for (; next < n_hi; ++next, ++bc) {
                    const int b = bc & 1;
                    if (!ready((p.ranks != nullptr ? b_fixed : b_full) + b, (uint32_t)((bc / 2) & 1), wait)) return;
                    if (bc >= 2 && !ready(d2_empty + b, (uint32_t)((bc / 2 - 1) & 1), wait)) return;
                    tc_fence_after();
                    for (int st = 0; st < steps; ++st) {
                        const uint64_t blk = (uint64_t)(st >> 2), in = (uint64_t)(2 * (st & 3));
                        const uint64_t bd = b0 + (uint64_t)((uint32_t)b * b_bytes >> 4) + blk * (b_block >> 4) + in;
                        for (int part_i = 0; part_i < parts; ++part_i)
                            mma_f16<1>(d2 + (uint32_t)(b * kLoraRows), bd,
                                       h0 + ((uint64_t)part_i * blocks + blk) * (h_block >> 4) + in, idesc,
                                       (uint32_t)(st | part_i));
                    }
                    gmm_commit<1>(b_empty + b);
                    gmm_commit<1>(d2_full + b);
                }
                gmm_commit<1>(&h_empty);
                open = false;
            };
            // a wait during which results are issued as they become ready
            auto wait_issuing = [&](uint64_t * bar, uint32_t parity) {
                uint32_t polls = 0;
                while (open) {
                    results(false);
                    if (mbar_test_wait(bar, parity) || ++polls == (1u << 20)) break;
                }
                if (polls == (1u << 20) && open) results(true);
                ok = ok && gmm_wait_one<1>(bar, parity, &abort_flag);
                return ok;
            };
            RingPos sum;                               // the accumulator of h in turn
            for (int t = unit; t < tiles && ok; t += units) {
                const LoraTile q = lora_tile(p, pre, t);
                if (q.rank == 0) continue;
                // (16 ranks sit in the first lanes of a 64-row MMA too, at half the shared memory reads)
                const uint32_t idesc = umma_idesc_f16(p.bf16 != 0, p.ra == 16 ? 64 : 128, (uint32_t)((q.cnt + 15) & ~15));
                int kc = k0;
                for (int sg = 0; sg < nseg && ok; ++sg, sum.next(kLoraSums)) {
                    const int first = kc, end = p.seg ? min(kc + p.seg, k1) : k1;
                    if (sum.round != 0) wait_issuing(d1_empty + sum.s, (sum.round - 1u) & 1u);
                    for (; kc < end && ok; ++kc, at.next(p.stages)) {
                        if (!wait_issuing(full + at.s, at.round & 1u)) break;
                        tc_fence_after();
                        const uint64_t off = (uint64_t)(((uint32_t)at.s * stage_bytes) >> 4);
#pragma unroll
                        for (int half = 0; half < 2; ++half)
#pragma unroll
                            for (int i = 0; i < kGmmK / 16; ++i)
                                mma_f16<1>(d1 + (uint32_t)(sum.s * kLoraRows), a0 + off + (uint64_t)(half * p.ra * 8 + 2 * i),
                                           x0 + off + (uint64_t)(half * (int)(kLoraXTile >> 4) + 2 * i), idesc,
                                           (uint32_t)((kc - first) | half | i));
                        gmm_commit<1>(empty + at.s);
                    }
                    if (ok) gmm_commit<1>(d1_full + sum.s);
                }
                if (!ok) break;
                if (open) results(true);
                if (!ok) break;
                last = q;
                next = n_lo;
                open = true;
                have_h = false;
                ++it;
            }
            if (ok && open) results(true);
            if (ok && it > 0) ok = gmm_wait_one<1>(&h_empty, (uint32_t)((it - 1) & 1), &abort_flag);
            if (!ok) {
                volatile int none = 0;
                gmm_commit<1>(&drained);
                gmm_wait_one<1>(&drained, 0, &none);
            }
        }
        __syncwarp();
    } else if (warp == 3) {
        // ------------------------------------------------------- B by TMA
        // and, where an adapter's rank ends inside a step of 16, B's columns
        // behind it cleared in shared memory: a zero in h does not silence a NaN
        int bc = 0, seen = 0, rank_was = 0;
        bool ok = true;
        auto fix = [&](int rank) {
            const int b = seen & 1;
            if (!gmm_wait<1>(b_full + b, (uint32_t)((seen / 2) & 1), &abort_flag)) return false;
            const int behind = rank < p.rank ? (rank + 15) & ~15 : rank;     // (behind the pool's rank TMA fills in zeros)
            if (rank < behind) {
                uint8_t * tile = bring + (uint32_t)b * b_bytes + (uint32_t)(rank >> 6) * b_block;
                for (int row = lane; row < 128; row += 32)
                    for (int r = rank; r < behind; ++r)
                        *reinterpret_cast<uint16_t *>(tile + lora_swizzle(row_bytes, row, (r & 63) >> 3) + (r & 7) * 2) = 0;
                fence_async_smem();
            }
            __syncwarp();
            if (lane == 0) gmm_arrive<1>(b_fixed + b);
            ++seen;
            return true;
        };
        for (int t = unit; t < tiles && ok; t += units) {
            const LoraTile q = lora_tile(p, pre, t);
            if (q.rank == 0) continue;
            for (int i = n_lo; i < n_hi && ok; ++i, ++bc) {
                const int b = bc & 1;
                if (bc >= 2) ok = gmm_wait<1>(b_empty + b, (uint32_t)((bc / 2 - 1) & 1), &abort_flag);
                if (!ok) break;
                if (elect_one()) {
                    const int nb = q.rank > 64 ? 2 : 1;
                    mbar_arrive_expect_tx(b_full + b, (uint32_t)nb * b_block);
                    for (int j = 0; j < nb; ++j)
                        tma_load_3d(bring + (uint32_t)b * b_bytes + (uint32_t)j * b_block, &p.bmap, j * 64, i * 128, q.g, b_full + b);
                }
                __syncwarp();
                // the tile before this one has had the time of a copy to land
                if (p.ranks != nullptr && bc > 0) ok = fix(rank_was);
                rank_was = q.rank;
            }
        }
        if (p.ranks != nullptr && ok && bc > 0) ok = fix(rank_was);
        for (int i = max(0, bc - 2); i < bc && ok; ++i) ok = gmm_wait<1>(b_empty + (i & 1), (uint32_t)((i / 2) & 1), &abort_flag);
        if (!ok) {
            volatile int none = 0;
            for (int i = max(0, bc - 2); i < bc; ++i) gmm_wait<1>(b_full + (i & 1), (uint32_t)((i / 2) & 1), &none);
        }
    } else {
        // ------------------------------------------------- h and results
        const int quad = warp & 3, ew = warp - 4;
        float * stage = staging + quad * (16 * 32);
        const int esz = p.out == GMM_F32 ? 4 : 2;
        const bool vec = ((reinterpret_cast<uintptr_t>(p.dst) | reinterpret_cast<uintptr_t>(p.base) | (uintptr_t)p.nbd |
                           (uintptr_t)p.nbb) & 15u) == 0;
        const bool row_pieces = (p.N * esz) % 16 == 0;         // whole 16-byte pieces
        int it = 0, bc = 0;
        RingPos sum;
        bool ok = true;
        for (int t = unit; t < tiles && ok; t += units) {
            const LoraTile q = lora_tile(p, pre, t);
            if (q.rank == 0) {
                if (p.copy) {
                    for (int j = ew * C + me; j < q.cnt; j += kLoraEpiWarps * C) {
                        bool bad = false;
                        const int row = lora_row(p, q.row0 + j, bad);
                        if (row < 0) continue;
                        if (esz == 4) lora_copy_row<float>(p, row, lane, 32);
                        else lora_copy_row<uint16_t>(p, row, lane, 32);
                    }
                }
                continue;
            }
            // what does not depend on h is on its way before h is
            bool bad = false;
            const int my = lane < q.cnt ? lora_row(p, q.row0 + lane, bad) : -1;
            const unsigned nans = __ballot_sync(0xffffffffu, bad);
            const float scale = p.scale != nullptr ? p.scale[q.g / p.n_as] : 1.0f;
            if (vec && row_pieces && ew == 0 && my >= 0 && n_lo < n_hi) {
                // base on its way into L2: lane's row, this CTA's columns (a megabyte at most)
                const uint32_t bytes = (uint32_t)min(min(n_hi * 128, p.N) - n_lo * 128, 1 << 18) * (uint32_t)esz;
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.base + (int64_t)my * p.nbb + (int64_t)n_lo * 128 * esz),
                             "r"(bytes)
                             : "memory");
            }
            // the partial h of this CTA's share of K: lanes are ranks, columns rows
            // (for f32 results in sums of 512 elements, added here with rounding)
            float own[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) own[i] = 0.0f;
            for (int sg = 0; sg < nseg && ok; ++sg, sum.next(kLoraSums)) {
                ok = gmm_wait<1>(d1_full + sum.s, sum.round & 1u, &abort_flag);
                if (!ok) break;
                tc_fence_after();
                if (quad * 32 < p.ra && k0 < k1) {
                    uint32_t v[32];
                    tmem_ld32(d1 + (uint32_t)(sum.s * kLoraRows) + ((uint32_t)quad << 21), v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) own[i] = __fadd_rn(own[i], __uint_as_float(v[i]));
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) gmm_arrive<1>(d1_empty + sum.s);
            }
            // (a release or acquire over the cluster also waits for the results' stores: one CTA alone does without)
            if (ok && it > 0) ok = C > 1 ? gmm_wait<2>(&part_free, (uint32_t)((it - 1) & 1), &abort_flag)
                                         : gmm_wait<1>(&part_free, (uint32_t)((it - 1) & 1), &abort_flag);
            if (!ok) break;
            if (const int r = quad * 32 + lane; r < p.ra) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (i < ((q.cnt + 15) & ~15)) part[i * p.ra + r] = own[i];
            }
            __syncwarp();
            if (C > 1) {
                arrive_all(&part_full, C);
                ok = gmm_wait<2>(&part_full, (uint32_t)(it & 1), &abort_flag);
            } else {
                if (lane == 0) gmm_arrive<1>(&part_full);
                ok = gmm_wait<1>(&part_full, (uint32_t)(it & 1), &abort_flag);
            }
            if (ok && it > 0) ok = gmm_wait<1>(&h_empty, (uint32_t)((it - 1) & 1), &abort_flag);
            if (!ok) break;
            // sum over the cluster in CTA order, scale, split, store as an MMA operand
            {
                const int per = p.ra / 8;                              // eight ranks per thread; a power of two <= 16
                const int rows16 = (q.cnt + 15) & ~15;
                const int items = rows16 * per;                        // a multiple of 32
                for (int i = ew * 32 + lane; i < items; i += kLoraEpiWarps * 32) {
                    const int row = i / per, r0 = (i - row * per) * 8;
                    float h[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) h[e] = 0.0f;
                    const float * from = part + row * p.ra + r0;
                    if (C == 1) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) h[e] = from[e];
                    } else {
                        // the loads of up to four CTAs together, the sums in CTA order
                        for (int c0 = 0; c0 < C; c0 += 4) {
                            float4 lo[4], hi[4];
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const int peer = min(c0 + c, C - 1);
                                lo[c] = ld_peer4(from, peer);
                                hi[c] = ld_peer4(from + 4, peer);
                            }
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                if (c0 + c >= C) break;
                                h[0] += lo[c].x; h[1] += lo[c].y; h[2] += lo[c].z; h[3] += lo[c].w;
                                h[4] += hi[c].x; h[5] += hi[c].y; h[6] += hi[c].z; h[7] += hi[c].w;
                            }
                        }
                    }
                    float big = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        h[e] = r0 + e < q.rank && row < q.cnt ? __fmul_rn(h[e], scale) : 0.0f;
                        const float size = fabsf(h[e]);
                        if (size < __int_as_float(0x7f800000)) big = fmaxf(big, size);
                    }
                    if (!p.bf16) {
                        // the row's largest finite |h| to [2^13, 2^14) (beside
                        // an infinity too: a finite h must not become another)
                        for (int m = 1; m < per; m <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, m));
                        const int e2 = big > 0.0f ? min(max((int)(__float_as_uint(big) >> 23) - 127 - 13, -126), 114) : 0;
                        const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
#pragma unroll
                        for (int e = 0; e < 8; ++e) h[e] = __fmul_rn(h[e], down);
                        if (r0 == 0) esc[row] = __uint_as_float((uint32_t)(127 + e2) << 23);
                    }
                    uint8_t * to = hbuf + (uint32_t)(r0 >> 6) * h_block + lora_swizzle(row_bytes, row, (r0 & 63) >> 3);
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        if (k >= lora_parts(p.bf16 != 0)) break;
                        uint4 v;
                        if (p.bf16) split_part<__nv_bfloat16>(h, v); else split_part<__half>(h, v);
                        *reinterpret_cast<uint4 *>(to + (uint32_t)k * blocks * h_block) = v;
                    }
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) gmm_arrive<1>(&h_full);
            if (C > 1) arrive_all(&part_free, C);
            else if (lane == 0) gmm_arrive<1>(&part_free);
            ok = gmm_wait<1>(&h_full, (uint32_t)(it & 1), &abort_flag);       // (every row's power of two)
            auto results = [&](auto base) {
                base.load(p, my, n_lo * 128 + quad * 32, vec);
                for (int nt = n_lo; nt < n_hi && ok; ++nt, ++bc) {
                    const int b = bc & 1, n0 = nt * 128 + quad * 32;
                    ok = gmm_wait<1>(d2_full + b, (uint32_t)((bc / 2) & 1), &abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    uint32_t v[32];
                    tmem_ld32(d2 + (uint32_t)(b * kLoraRows) + ((uint32_t)quad << 21), v);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) gmm_arrive<1>(d2_empty + b);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (half * 16 >= q.cnt) break;
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float f = __uint_as_float(v[half * 16 + i]);
                            if (!p.bf16) f = __fmul_rn(f, esc[half * 16 + i]);
                            if ((nans >> (half * 16 + i)) & 1u) f = kNan;
                            stage[i * 32 + lane] = f;
                        }
                        __syncwarp();
                        base.add(p, stage, half, my, n0, vec);
                    }
                    if (nt + 1 < n_hi) base.load(p, my, n0 + 128, vec);
                }
            };
            if (p.out == GMM_F32) results(LoraBase<float>{});
            else if (p.out == GMM_BF16) results(LoraBase<__nv_bfloat16>{});
            else results(LoraBase<__half>{});
            ++it;
        }
    }
    tc_fence_before();
    if (C > 1) cluster_sync_all(); else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        gmm_tmem_free<1>(tbase, kLoraTmem);
    }
}

}  // namespace gx
