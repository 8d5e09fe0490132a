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
//
// A persistent kernel; per CTA a ring of stages of 64 elements of K (128-byte
// swizzled rows): one warp copies the matrix tiles (and rows that lie in
// place) by TMA, up to four warps gather other rows by tile::gather4, one
// thread issues the MMAs, four or eight warps read the accumulators, apply
// the activation and write 16-byte pieces by way of shared memory. Bounds and
// choices, as measured on a B200 (1617 TFLOP/s, 6552 GB/s measured peaks; calls
// in a row on one set of inputs, a few percent faster than on changing ones):
//   - Few rows per expert: HBM. Gated, 19 tokens over 64 experts (hidden 2048,
//     intermediate 1024): 50 us, 5.5 TB/s. Tiles of 32 rows leave room for a
//     ring of ten stages. A last round of tiles that would leave most SMs idle
//     is shared by clusters that split K (gated, 2880 x 2880, 4 experts: 180
//     tiles on 148 SMs, 33 us without, 29 with).
//   - Long groups: the tensor cores. CTA pairs (256 x 256 tiles): 32768 rows,
//     K 4096, N 1536 take 300 us in place (1371 TFLOP/s) and 334 us gathered. A
//     single CTA's 128 x 256 tile would need 96 bytes a cycle of L2, a pair's
//     needs 64; the same shape took 495 us on single CTAs. With f32 results it
//     takes 400 us: four warps add the accumulators up (512 elements of K each)
//     and stage twice the bytes.
//   - Gated pairs keep 128 gate and 128 up rows per CTA against the same rows
//     (both accumulators fill TMEM, nothing takes turns): a copied row is used
//     twice, which gather4 (24 cycles per four rows) needs. 8192 tokens, 8
//     experts each, K 4096, N 1536: 1128 us against 1244 with 64 + 64 rows and
//     two accumulators in turn, 384 against 461 at K 1024 (both since a little
//     faster: 1110 us, 1485 TFLOP/s, and 368). At 128 registers a thread 20
//     bytes of it spill. In the case of 128 experts (1.65 PFLOP) a pass takes
//     1470 us at 1965 MHz; back to back the board's power limit holds the SMs at
//     1365 MHz (990 W) and a pass takes 1630. Spreading short groups' tiles
//     among the long ones' changed nothing (1514 us for 1506).
//   - The thread that issues copies or MMAs is chosen by elect.sync: with
//     `lane == 0` a stage took 768 cycles, with it 590, of 512 for its MMAs.
//   - Gathering by cp.async needs twelve warps (the fence that shows a stage
//     to the tensor cores waits for all of a warp's copies) and reached 1043
//     TFLOP/s where gather4 reaches 1234.
//
// With 4-bit weights (SRC; Q4_0 and Q4_1 blocks) eight warps make the matrix
// tiles instead: w = d (q - 8) or d q + m as two (Q4_1, BF16 rows, f32 results: three)
// 16-bit values, each the rest rounded, one MMA per part into the same sums.
//   - Two parts: results are as far from 64 bits as sums of exact products (f32
//     6e-7, BF16 1.7e-3, which is the rounding of the result). One part, a weight
//     rounded to 8 or 11 bits, is faster (gated 2048 tokens, 128 experts, 4096 x 1536:
//     818 us for 956) but leaves 16-bit results 1.7 times as far.
//   - What bounds it: the MMAs of both parts, 1024 cycles a chunk of 64 elements, and
//     hardly less the warps that make tiles, 900 to 1200. 2048 rows, 4096 x 14336: 332
//     us, 724 TFLOP/s of products, 1450 with both parts; 512 rows keep the tensor pipe
//     72 % busy. Short groups pay for whole tiles of weights: 1031 tokens x 8 of 64
//     experts, 1024 x 2048, f32 results, 141 us and 36 more for those of up to 24 rows.
//   - Tried, no gain: twelve warps in three fours, a register split by setmaxnreg
//     (spills), blocks loaded straight into registers (278 us where boxes took 220).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gx_grouped_plan.h"
#include "gx_tc.cuh"
#include "gx_wait.cuh"

namespace gx {

enum : int { GMM_F32 = 0, GMM_F16 = 1, GMM_BF16 = 2 };

struct GmmParams {
    CUtensorMap wmap;         // W (or G): [K, N, G], boxes 64 x gmm_out_rows
    CUtensorMap umap;         // U
    CUtensorMap xmap;         // x: [K, rows], boxes 64 x box, 64 x 1 for gathers
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
    int32_t nt;               // rows of a group per tile (multiple of 32)
    int32_t stages;
    int32_t box;              // rows of one TMA box of x in place (divides nt / CTAs)
    int32_t mt;               // tiles of the matrix rows
    int32_t most;             // tiles of nt rows that groups can have
    int32_t split;            // CTAs of a cluster that share K (single CTAs with nt = 32 only)
    int32_t seg;              // chunks that one accumulator sums (0: all)
    int32_t acc;              // TMEM columns of an accumulator
    // 4-bit weights (SRC != 0): the matrices in place of the maps
    const uint8_t * w0;       // W (or G)
    const uint8_t * w1;       // U
    int64_t nb01, nb02;
    int32_t parts;            // 16-bit parts that a weight is made of
    int32_t lo;               // rows of the shortest group that the launch is for
    int32_t boxes;            // rows on 16 bytes: wmap and umap are maps of the blocks, [words of a row, N, G]
};

// Where the matrix tiles come from: 16-bit weights by TMA, or blocks of 4-bit
// ones, which warps of their own turn into tiles of the rows' type
enum : int { GMM_TILES = 0, GMM_Q4_0_F16 = 1, GMM_Q4_0_BF16 = 2, GMM_Q4_1_F16 = 3, GMM_Q4_1_BF16 = 4 };

// ------------------------------------------------------------ PTX helpers

template <int CTAS>
__device__ __forceinline__ void gmm_tmem_alloc(uint32_t * dst, uint32_t cols) {
    if constexpr (CTAS == 1) {
        tmem_alloc(dst, cols);
        tmem_relinquish();
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void gmm_tmem_free(uint32_t addr, uint32_t cols) {
    if constexpr (CTAS == 1) tmem_dealloc(addr, cols);
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}

// D[tmem] (+)= A x B^T, f16 or bf16 operands, f32 accumulators, one thread (of
// the leading CTA; a pair's A is 2 x 128 rows and each CTA holds half of B's rows)
template <int CTAS>
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
    if constexpr (CTAS == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum)
            : "memory");
}

// the barrier (in both CTAs of a pair) arrives once this thread's MMAs so far are done
template <int CTAS>
__device__ __forceinline__ void gmm_commit(uint64_t * bar) {
    if constexpr (CTAS == 1) mma_commit(bar);
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
            "h"((uint16_t)3)
            : "memory");
}

// instruction descriptor of kind::f16: f32 accumulator, A and B of one type, both K-major
__host__ __device__ constexpr uint32_t umma_idesc_f16(bool bf16, uint32_t M, uint32_t N) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((N >> 3) << 17) | ((M >> 4) << 24);
}

// TMA tiles into this CTA's shared memory. In a pair the bytes are counted on
// the leading CTA's barrier: bit 24 of a shared-memory address tells the
// CTAs of a pair apart, and cta_group::2 lets a copy signal its peer.
constexpr uint32_t kLeaderMask = 0xFEFFFFFFu;

template <int CTAS>
__device__ __forceinline__ void gmm_tma_3d(void * dst, const CUtensorMap * map, int x, int y, int z, uint64_t * bar) {
    if constexpr (CTAS == 1) tma_load_3d(dst, map, x, y, z, bar);
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
            "%4}], [%5];" ::"r"(smem_u32(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar) & kLeaderMask)
            : "memory");
}
template <int CTAS>
__device__ __forceinline__ void gmm_tma_2d(void * dst, const CUtensorMap * map, int x, int y, uint64_t * bar) {
    if constexpr (CTAS == 1)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                smem_u32(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
            "[%4];" ::"r"(smem_u32(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar) & kLeaderMask)
            : "memory");
}

// arrive on the same barrier of every CTA of the cluster (lane c of the warp: CTA c)
__device__ __forceinline__ void arrive_all(uint64_t * bar, int ctas) {
    const int lane = threadIdx.x & 31;
    if (lane < ctas)
        asm volatile(
            "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, %1;\n\t"
            "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [r];\n\t}" ::"r"(smem_u32(bar)),
            "r"(lane)
            : "memory");
}
// arrive on the barrier of CTA `cta`, and a value of its shared memory
__device__ __forceinline__ void arrive_at(uint64_t * bar, int cta) {
    asm volatile(
        "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, %1;\n\t"
        "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [r];\n\t}" ::"r"(smem_u32(bar)),
        "r"(cta)
        : "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void * p, int cta) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(cta));
    return r;
}
__device__ __forceinline__ float ld_peer(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// 32 consecutive columns of this thread's TMEM lane, to be waited for (the
// second call only ties the registers to the wait)
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32_end(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                   "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])::"memory");
    asm volatile("" : "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                 "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])::"memory");
}

// 32 consecutive columns of this thread's TMEM lane, written
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
    tmem_wait_st();
}

// four rows of a map with boxes of one row (no multicast: this GPU's own memory)
template <int CTAS>
__device__ __forceinline__ void gmm_gather4(void * dst, const CUtensorMap * map, int x, int r0, int r1, int r2, int r3,
                                            uint64_t * bar) {
    if constexpr (CTAS == 1)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
            "%4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(smem_u32(bar))
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, "
            "{%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(smem_u32(bar) & kLeaderMask)
            : "memory");
}

// arrive on the barrier of the leading CTA: this CTA's reads of TMEM are done
// (they are ordered by the tcgen05 fences; a release over the cluster would
// also wait for the results' stores to reach L2)
template <int CTAS>
__device__ __forceinline__ void gmm_arrive(uint64_t * bar) {
    if constexpr (CTAS == 1)
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
    else
        asm volatile(
            "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, 0;\n\t"
            "mbarrier.arrive.release.cta.shared::cluster.b64 _, [r];\n\t}" ::"r"(smem_u32(bar))
            : "memory");
}

// one thread of a whole warp (the compiler then knows that values of the
// branch belong to one thread, as the TMA and MMA operands need)
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// a value's agreement over the two warps that share a named barrier
__device__ __forceinline__ bool pair_agrees(int id, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(id)
        : "memory");
    return r != 0;
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

// pre[g] = tiles of nt rows in the groups before g (G + 1 values), by the
// whole block; rows(g) are the rows of group g. Groups that do not overlap have
// at most `most` tiles; borders that name more (sums stop there, so none wraps
// round) are reported, and the launch has no tiles.
template <typename F>
__device__ __forceinline__ void tile_prefix(int32_t * pre, int32_t * wsum, int G, int nt, int most, F && rows) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = blockDim.x;
    const int per = (G + n - 1) / n;
    const int g0 = min(tid * per, G), g1 = min(g0 + per, G);
    const int cap = most + 1;                   // (2^26 + 8194 at most)
    int sum = 0;
    for (int g = g0; g < g1; ++g) {
        const int2 r = rows(g);
        pre[g] = sum;
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
    for (int g = g0; g < g1; ++g) pre[g] += before;
    if (tid == n - 1) {
        const bool over = before + sum > most;
        if (over) record_error(GX_DEVERR_DOMAIN);
        pre[G] = over ? 0 : before + sum;
    }
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

// tile t of the launch: the tiles of the matrix run fastest, so that CTAs at
// work together read the same rows and one expert's weights (m0: its first
// matrix row, `rows` per tile)
template <int ROUND, int SRC = GMM_TILES>
__device__ __forceinline__ GmmTile gmm_tile(const GmmParams & p, const int32_t * pre, int t, int rows) {
    GmmTile r;
    const int tt = t / p.mt;
    r.m0 = (t - tt * p.mt) * rows;
    r.g = tile_group(pre, p.G, tt);
    const bool all = SRC != GMM_TILES && p.offsets == nullptr;          // (one matrix for all rows)
    const int lo = all ? 0 : p.offsets[r.g], hi = all ? p.n_rows : p.offsets[r.g + 1];
    // a group's tiles are of one size, rather than full ones and a rest
    const int n = pre[r.g + 1] - pre[r.g];
    const int size = ((hi - lo - 1) / n + ROUND) / ROUND * ROUND;
    r.row0 = lo + (tt - pre[r.g]) * size;
    r.cnt = min(size, hi - r.row0);
    return r;
}

// fours of rows that gathering warp w copies of a CTA's n
__device__ __forceinline__ int gather_quads(int n, int w) { return max(1, (min(32, n - w * 32) + 3) >> 2); }

// y row of grouped row j, -1 to skip it (no such row); nan: its x row does not exist
// (o: order[j], where it is read at all)
template <typename P>
__device__ __forceinline__ int gmm_dst_row(const P & p, int j, int o, bool & nan) {
    if (p.gather == 0 && p.scatter == 0) return j;
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

// e^x / 4 without branches: x is clamped to where the quarter leaves the normal
// range (n = 130 makes the scale infinite) or is nothing beside 1, n = x log2 e
// to nearest, r = x - n ln 2 with ln 2 in two parts (Cody and Waite, 1980), e^r
// by its Taylor polynomial; within 2 f32 steps in between
__device__ __forceinline__ float gmm_quarter_exp(float x) {
    x = fminf(fmaxf(x, -85.0f), 90.25f);
    const float t = __fmaf_rn(x, 1.44269502162933349609375f, 12582912.0f);
    const float n = __fsub_rn(t, 12582912.0f);
    float r = __fmaf_rn(-n, 0.693145751953125f, x);
    r = __fmaf_rn(-n, 1.428606765330187045e-06f, r);
    float q = __fmaf_rn(r, 1.98412701138295233249664306640625e-04f, 1.3888889225199818611145019531250e-03f);
    q = __fmaf_rn(q, r, 8.3333337679505348205566406250000e-03f);
    q = __fmaf_rn(q, r, 4.1666667908430099487304687500000e-02f);
    q = __fmaf_rn(q, r, 1.6666667163372039794921875000000e-01f);
    q = __fmaf_rn(q, r, 0.5f);
    q = __fmaf_rn(q, r, 1.0f);
    q = __fmaf_rn(q, r, 1.0f);
    return __fmul_rn(q, __uint_as_float((__float_as_uint(t) + 125u) << 23));
}

// The activation on f32 sums. The quotient is CUDA's fast division (2 steps):
// the sums are not those of the bit-exact formats anyway, and a full division
// per value kept the epilogue behind the tensor cores. It gives zero for a
// divisor above 2^126, hence a quarter of both sides: 1 + e^z then stays below
// that wherever e^z is finite. FAST: CUDA's fast exp as well, about |x| f32
// steps off, for results of 16 bits, whose rounding is hundreds of times that
// (8192 tokens, 8 experts each, K 1024: 367 us, with the polynomial 384).
template <bool FAST>
__device__ __forceinline__ float gmm_sigmoid_times(float x, float z) {       // x / (1 + e^z)
    const float y = FAST ? __fmaf_rn(0.25f, __expf(z), 0.25f) : __fadd_rn(0.25f, gmm_quarter_exp(z));
    return __fdividef(__fmul_rn(0.25f, x), y);
}
template <bool OAI, bool FAST, typename P>
__device__ __forceinline__ float gmm_act(const P & p, float g, float u) {
    if (!OAI) return __fmul_rn(gmm_sigmoid_times<FAST>(g, -g), u);
    const float x = p.limit < g ? p.limit : g;
    const float y = u < -p.limit ? -p.limit : (p.limit < u ? p.limit : u);
    return __fmul_rn(gmm_sigmoid_times<FAST>(x, __fmul_rn(p.alpha, -x)), __fadd_rn(y, 1.0f));
}
// of N values at once: g becomes the result (the choices stay outside the
// loop, so that the values' chains of operations overlap)
template <bool OAI, bool FAST, int N, typename P>
__device__ __forceinline__ void gmm_act_each(const P & p, float (&g)[N], const float (&u)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = gmm_act<OAI, FAST>(p, g[i], u[i]);
}
template <int N, typename P>
__device__ __forceinline__ void gmm_act_all(const P & p, float (&g)[N], const float (&u)[N]) {
    if (p.out == GMM_F32) {
        if (p.act == 0) gmm_act_each<false, false, N>(p, g, u);
        else gmm_act_each<true, false, N>(p, g, u);
    } else {
        if (p.act == 0) gmm_act_each<false, true, N>(p, g, u);
        else gmm_act_each<true, true, N>(p, g, u);
    }
}

// position in the ring of stages: stage, and how often the ring was gone round
struct RingPos {
    int s = 0;
    uint32_t round = 0;
    __device__ __forceinline__ void next(int stages) {
        if (++s == stages) {
            s = 0;
            ++round;
        }
    }
    __device__ __forceinline__ void skip(int n, int stages) {
        s += n;
        round += (uint32_t)(s / stages);
        s %= stages;
    }
};

// 32 (or 16) columns of a warp's 32 matrix rows, staged as [column][row], to
// their result rows: 16-byte pieces where rows allow them (`vec`), element by
// element at a ragged edge. `my` is lane i's result row of column i.
template <typename T, int COLS>
__device__ __forceinline__ void store_rows(const GmmParams & p, const uint8_t * stage, int my, int n0, bool vec) {
    constexpr int kPer = 16 / (int)sizeof(T);                 // elements of a piece
    constexpr int kLanes = 32 / kPer;                         // lanes of a row
    const int lane = threadIdx.x & 31, sub = lane % kLanes;
    const int n = n0 + sub * kPer;
#pragma unroll
    for (int c = 0; c < COLS; c += 32 / kLanes) {
        const int col = c + lane / kLanes;
        const int row = __shfl_sync(0xffffffffu, my, col);
        if (row < 0) continue;
        const uint4 v = *reinterpret_cast<const uint4 *>(stage + (uint32_t)(col * 32 + sub * kPer) * sizeof(T));
        T * out = reinterpret_cast<T *>(p.dst + (int64_t)row * p.nbd1) + n;
        if (vec && n + kPer <= p.N) *reinterpret_cast<uint4 *>(out) = v;
        else {
            const T * e = reinterpret_cast<const T *>(&v);
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (n + i < p.N) out[i] = e[i];
        }
    }
}

template <typename T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ float round_to<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// lane's COLS values, rounded, through the warp's staging area to the result rows
template <typename T, int COLS>
__device__ __forceinline__ void put_rows(const GmmParams & p, uint8_t * stage, const float (&v)[COLS], int my, int n0, bool vec) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < COLS; ++i) reinterpret_cast<T *>(stage)[i * 32 + lane] = round_to<T>(v[i]);
    __syncwarp();
    store_rows<T, COLS>(p, stage, my, n0, vec);
}
template <int COLS>
__device__ __forceinline__ void put_rows_as(const GmmParams & p, uint8_t * stage, const float (&v)[COLS], int my, int n0, bool vec) {
    if (p.out == GMM_F32) put_rows<float, COLS>(p, stage, v, my, n0, vec);
    else if (p.out == GMM_BF16) put_rows<__nv_bfloat16, COLS>(p, stage, v, my, n0, vec);
    else put_rows<__half, COLS>(p, stage, v, my, n0, vec);
}

// Eight weights as `parts` sums of 16-bit values: 16 bytes of each part's tile
__device__ __forceinline__ void q4_store(uint32_t to, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
template <bool BF16>
__device__ __forceinline__ uint32_t q4_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// `one`: 1 in both halves (a sum as a product with 1)
template <bool BF16>
__host__ __device__ constexpr uint32_t q4_one() {
    return BF16 ? 0x3F803F80u : 0x3C003C00u;
}

// d (q - 8) for eight codes in the bytes of two words' low (or high) halves, two
// 16-bit values at a time. q - 8 has four bits, d eleven: F16 rounds their product
// once, and the rest is a 16-bit value too. BF16 takes d in two parts of eight and
// three bits; q - 8 times the second is exact, so a product and a sum round once.
template <bool BF16>
struct Q4Scale {
    uint32_t hi, lo;
    __device__ __forceinline__ Q4Scale(__half d) {
        if constexpr (BF16) {
            const __nv_bfloat16 h = __float2bfloat16_rn(__half2float(d));
            const __nv_bfloat162 a = __halves2bfloat162(h, h);
            const __nv_bfloat162 b = __float2bfloat162_rn(__fsub_rn(__half2float(d), __bfloat162float(h)));
            hi = *reinterpret_cast<const uint32_t *>(&a);
            lo = *reinterpret_cast<const uint32_t *>(&b);
        } else {
            const __half2 a = __halves2half2(d, d);
            hi = *reinterpret_cast<const uint32_t *>(&a);
            lo = 0u;
        }
    }
};
// the first part of a pair, q - 8 being left in q and its product with d.lo in t
template <bool BF16>
__device__ __forceinline__ uint32_t q4_first_part(uint32_t & q, uint32_t & t, const Q4Scale<BF16> & d) {
    // 16 + q - 24 (BF16), 64 + q - 72 (F16)
    q = q4_fma<BF16>(q, q4_one<BF16>(), BF16 ? 0xC1C0C1C0u : 0xD480D480u);
    t = BF16 ? q4_fma<BF16>(q, d.lo, 0x80008000u) : 0x80008000u;
    return q4_fma<BF16>(q, d.hi, t);
}
// and what is left of it
template <bool BF16>
__device__ __forceinline__ uint32_t q4_second_part(uint32_t v, uint32_t q, uint32_t t, const Q4Scale<BF16> & d) {
    v = q4_fma<BF16>(q, d.hi, v ^ 0x80008000u);
    return BF16 ? q4_fma<BF16>(t, q4_one<BF16>(), v) : v;
}
// bytes of codes (q << 3 | 0x80, or q << 4) as pairs of 16 + q (BF16) or 64 + q (F16)
template <bool BF16>
__device__ __forceinline__ void q4_pairs(uint32_t word, bool high, uint32_t & a, uint32_t & b) {
    uint32_t v;
    if constexpr (BF16) v = ((high ? word >> 1 : word << 3) & 0x78787878u) | 0x80808080u;
    else v = (high ? word : word << 4) & 0xF0F0F0F0u;
    constexpr uint32_t top = BF16 ? 0x41414141u : 0x54545454u;
    a = __byte_perm(v, top, 0x4140);
    b = __byte_perm(v, top, 0x4342);
}

// Four bytes of codes as f32: 16 + q, the code in the upper bits of the mantissa
// (bytes of 0x80 | q << 3 into the third byte of 0x41......)
__device__ __forceinline__ void q4_spread(uint32_t bytes, float * f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(bytes, 0x41u, 0x4055u + 0x100u * (uint32_t)i));
}
// Eight weights from f32, each part the rest rounded
template <bool BF16>
__device__ __forceinline__ void q4_put(float (&w)[8], uint32_t to, int parts) {
    for (int part = 0; part < parts; ++part, to += kGmmATile) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(w[2 * i], w[2 * i + 1]);
                v[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __half2 h = __floats2half2_rn(w[2 * i], w[2 * i + 1]);
                v[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        q4_store(to, v);
        if (part + 1 == parts) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 h;
            if constexpr (BF16) h = make_float2(__uint_as_float(v[i] << 16), __uint_as_float(v[i] & 0xFFFF0000u));
            else h = __half22float2(*reinterpret_cast<const __half2 *>(&v[i]));
            w[2 * i] = __fsub_rn(w[2 * i], h.x);
            w[2 * i + 1] = __fsub_rn(w[2 * i + 1], h.y);
        }
    }
}

// NaN in place of what a warp gave up: 32 matrix rows from m on of tile t and those behind it
template <int ROUND, int SRC>
__device__ __noinline__ void gmm_fill_nan(const GmmParams & p, const int32_t * pre, int t, int units, int tiles, int rows, int m) {
    for (; t < tiles; t += units) {
        const GmmTile q = gmm_tile<ROUND, SRC>(p, pre, t, rows);
        const int n = q.m0 + m + (int)(threadIdx.x & 31);
        for (int j = q.row0; j < q.row0 + q.cnt && n < p.N; ++j) {
            bool nan = false;
            const int to = gmm_dst_row(p, j, p.gather != 0 || p.scatter != 0 ? p.order[j] : 0, nan);
            if (to >= 0) store_out(p.dst + (int64_t)to * p.nbd1, n, kNan, p.out);
        }
    }
}

template <int CTAS, int MODE, int SRC>
__global__ void __launch_bounds__(SRC != GMM_TILES ? gmm_q4_threads(MODE) : gmm_threads(MODE), 1)
    k_gmm(const __grid_constant__ GmmParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[kGmmMaxStages], empty[kGmmMaxStages], acc_full[2], acc_empty[2], part_full, part_free[2], drained;
    __shared__ uint32_t tslot;
    __shared__ int4 gather_mem[SRC != GMM_TILES ? 3 * kGmmQ4Quads : kGmmGatherWarps * 8];
    constexpr int kQ4 = SRC != GMM_TILES ? kGmmQ4Warps : 0;              // warps that make matrix tiles
    constexpr int kGather = SRC != GMM_TILES ? kGmmQ4GatherWarps : kGmmGatherWarps;
    __shared__ uint64_t raw_full[kQ4 ? 4 : 1][kGmmQ4Stages], raw_empty[kQ4 ? 4 : 1][kGmmQ4Stages];
    __shared__ int32_t wsum[gmm_threads(MODE) / 32 + kQ4];
    __shared__ int abort_flag;
    int32_t * gather_rows = reinterpret_cast<int32_t *>(gather_mem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = CTAS == 1 ? 0 : (int)(blockIdx.x & 1);              // CTA of the pair; 0 leads
    const int split = CTAS == 1 ? p.split : 1;
    const int me = CTAS == 1 ? (int)blockIdx.x % split : 0;             // share of K
    constexpr bool GLU = MODE == GMM_GLU;
    constexpr int kBufs = MODE == GMM_DUAL ? 1 : 2;                      // accumulators that take turns
    constexpr int kEpi = gmm_epi_warps(MODE);
    const uint32_t kABytes = SRC != GMM_TILES ? (uint32_t)p.parts * kGmmATile : gmm_a_bytes(MODE);
    uint8_t * ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t stage_bytes = kABytes + (uint32_t)(p.nt / CTAS) * 128u;
    uint8_t * raw = ring + (uint32_t)p.stages * stage_bytes;             // 4-bit weights: the rings of blocks
    uint8_t * staging = raw + (SRC != GMM_TILES ? gmm_q4_raw(SRC >= GMM_Q4_1_F16) : 0u);
    float * xchg = reinterpret_cast<float *>(staging + kGmmStaging);
    float * part = xchg + (GLU ? kGmmXchg / 4 : 0u);                     // [2][nt][128] partial sums of a shared tile
    int32_t * pre = reinterpret_cast<int32_t *>(part + (split > 1 ? 2 * p.nt * kGmmRows : 0));
    constexpr int kOut = gmm_out_rows(MODE);                             // result rows of a CTA's tile
    constexpr int kRound = 16 * CTAS;                                    // MMA N: a multiple of this

    if (tid == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(full + i, SRC != GMM_TILES ? CTAS * ((p.gather ? 1 + kGmmQ4GatherWarps : 1) + kQ4 / 2) : 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + i, 1);
            mbar_init(acc_empty + i, kEpi * CTAS);
        }
        for (int i = 0; i < (kQ4 ? 4 * kGmmQ4Stages : 0); ++i) {
            mbar_init(&raw_full[0][0] + i, 1);
            mbar_init(&raw_empty[0][0] + i, 2);
        }
        mbar_init(&part_full, (uint32_t)(kEpi * split));
        for (int i = 0; i < 2; ++i) mbar_init(part_free + i, kEpi);
        mbar_init(&drained, 1);
        abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) gmm_tmem_alloc<CTAS>(&tslot, 512);
    if constexpr (SRC != GMM_TILES) {
        griddep_launch_dependents();
        griddep_wait();
    }
    tile_prefix(pre, wsum, p.G, p.nt, p.most, [&](int g) {
        if (SRC != GMM_TILES && p.offsets == nullptr) return make_int2(0, p.n_rows);
        const int2 r = group_rows_of(p.offsets, g, p.n_rows);
        return SRC != GMM_TILES && r.y - r.x < p.lo ? make_int2(0, 0) : r;
    });
    tc_fence_before();
    if (CTAS * split == 1) __syncthreads(); else cluster_sync_all();
    tc_fence_after();
    const uint32_t tbase = tslot;
    const int tiles = pre[p.G] * p.mt;
    const int nk = (p.K + kGmmK - 1) / kGmmK;
    // The tiles in turn: whole ones, a CTA (or pair) each, and, when few are
    // left for the last round, those by all CTAs of a cluster that share K.
    const int unit = (int)blockIdx.x / CTAS, units = (int)gridDim.x / CTAS;
    const int cid = (int)blockIdx.x / (CTAS * split), clusters = (int)gridDim.x / (CTAS * split);
    int whole = tiles;
    if (split > 1) {
        const int rest = tiles % units;
        // (about three chunks of time go into a shared tile's exchange; shared
        // and whole, gated: 180 tiles of 45 chunks 28.5 and 32.9 us, 128 of 32
        // chunks 19.1 and 16.3, 320 of 112 chunks 87.5 and 100.6)
        if ((rest + clusters - 1) / clusters * (nk / split + 3) < nk) whole = tiles - rest;
    }
    struct Work {
        int t;
        bool shared;
    };
    auto start = [&] { return unit < whole ? Work{unit, false} : Work{whole + cid, true}; };
    auto advance = [&](Work & w) {
        w.t += w.shared ? clusters : units;
        if (!w.shared && w.t >= whole) w = Work{whole + cid, true};
    };
    auto first_chunk = [&](const Work & w) { return w.shared ? nk * me / split : 0; };
    auto end_chunk = [&](const Work & w) { return w.shared ? nk * (me + 1) / split : nk; };
    const int gathering = p.gather ? (p.nt / CTAS + 31) / 32 : 0;        // warps that gather

    if (SRC != GMM_TILES && (warp == 0 || (warp >= 2 && warp < 2 + kGmmQ4GatherWarps))) {
        // --------------------------------------- rows, beside 4-bit weights
        // Rows in place by one thread, or gathered by three warps, which take the
        // fours of a CTA's rows in turn. Each arrives at every stage, with rows or
        // without: a stage that did not wait for it could go round the ring twice
        // before it looks, and the parity of its barrier would then say the opposite
        // (this timed out once, with groups of a few rows among long ones).
        const int gi = warp == 0 ? 0 : warp - 1;
        if (gi == 0 || p.gather != 0) {
            int32_t * rows = gather_rows + gi * (4 * kGmmQ4Quads);
            RingPos at;
            bool ok = true;
            int c = 0, done = 0;       // chunks started; chunks whose stage was handed back
            for (Work w = start(); w.t < tiles && ok; advance(w)) {
                const GmmTile q = gmm_tile<kRound, SRC>(p, pre, w.t, kOut * CTAS);
                const int half = ((q.cnt + kRound - 1) / kRound * kRound) / CTAS;      // rows of x per CTA
                auto rows_of = [&](int r) { return max(0, min(half, q.cnt - r * half)); };
                const int n = rows_of(rank), r0 = q.row0 + rank * half, all_quads = (n + 3) >> 2;
                const int quads = p.gather ? (all_quads - gi + 2) / 3 : 0, boxes = p.gather ? 0 : (n + p.box - 1) / p.box;
                uint32_t bytes = 0;
                for (int r = 0; r < CTAS; ++r)
                    bytes += p.gather ? (uint32_t)((rows_of(r) + 3) >> 2) * 512u : (uint32_t)((rows_of(r) + p.box - 1) / p.box) * (p.box * 128u);
                __syncwarp();
                for (int i = lane; i < 4 * quads; i += 32) {
                    // (rows behind the last repeat it)
                    const int o = p.order[r0 + min(4 * (gi + 3 * (i >> 2)) + (i & 3), n - 1)];
                    int row = o / p.gather;
                    if (o < 0 || row >= p.x_rows) {
                        record_error(GX_DEVERR_DOMAIN);
                        row = 0;
                    }
                    rows[i] = row;
                }
                __syncwarp();
                if (elect_one()) {
                    // (the rows in registers, the copies one behind the other: read in a loop they took 85 cycles each)
                    int4 of[kGmmQ4Quads];
#pragma unroll
                    for (int i = 0; i < kGmmQ4Quads; ++i) of[i] = *reinterpret_cast<const int4 *>(rows + 4 * i);
                    RingPos on = at;
                    for (int kc = 0; kc < nk; ++kc, ++c, on.next(p.stages)) {
                        if (on.round != 0) {
                            ok = gmm_wait_one<CTAS>(empty + on.s, (on.round - 1u) & 1u, &abort_flag);
                            if (!ok) break;
                            ++done;
                        }
                        uint64_t * bar = full + on.s;
                        if (rank == 0 && gi == 0) mbar_arrive_expect_tx(bar, bytes);
                        else gmm_arrive<CTAS>(bar);
                        uint8_t * to = ring + (uint32_t)on.s * stage_bytes + kABytes;
                        if (boxes) gmm_tma_2d<CTAS>(to, &p.xmap, kc * kGmmK, r0, bar);      // (half a tile's rows: one box)
#pragma unroll
                        for (int i = 0; i < kGmmQ4Quads; ++i)
                            if (i < quads)
                                gmm_gather4<CTAS>(to + (gi + 3 * i) * 512, &p.xmap, kc * kGmmK, of[i].x, of[i].y, of[i].z, of[i].w, bar);
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                at.skip(nk, p.stages);
            }
            if (gi == 0 && (c = __reduce_max_sync(0xffffffffu, c)) > 0) {
                done = __reduce_max_sync(0xffffffffu, done);
                // (the issuer's commits arrive in both CTAs of a pair: the last ones too, before either leaves)
                for (int i = max(0, c - p.stages); i < c && ok; ++i)
                    ok = gmm_wait<CTAS>(empty + i % p.stages, (uint32_t)((i / p.stages) & 1), &abort_flag);
                if (!ok && rank == 0) {
                    // copies in flight land before the CTA leaves
                    volatile int none = 0;
                    for (int i = done; i < c; ++i) gmm_wait<CTAS>(full + i % p.stages, (uint32_t)((i / p.stages) & 1), &none);
                }
            }
        }
    } else if (warp == 0) {
        // ------------------------------------------- weights, rows in place
        if (elect_one()) {
            int c = 0, done = 0;       // chunks started; chunks whose stage was handed back
            RingPos at;
            bool ok = true;
            for (Work w = start(); w.t < tiles && ok; advance(w)) {
                const GmmTile q = gmm_tile<kRound, SRC>(p, pre, w.t, kOut * CTAS);
                const int k0 = first_chunk(w), k1 = end_chunk(w);
                const int m0 = q.m0 + rank * kOut;
                const int half = ((q.cnt + kRound - 1) / kRound * kRound) / CTAS;      // rows of x per CTA
                const int r0 = q.row0 + rank * half;
                uint32_t bytes = (uint32_t)CTAS * kABytes;
                int boxes = 0;
                for (int r = 0; r < CTAS; ++r) {
                    const int n = max(0, min(half, q.cnt - r * half));
                    if (p.gather) {
                        for (int w = 0; w < gathering; ++w) bytes += (uint32_t)gather_quads(n, w) * 512u;
                    } else {
                        const int b = (n + p.box - 1) / p.box;
                        bytes += (uint32_t)b * (p.box * 128u);
                        if (r == rank) boxes = b;
                    }
                }
                for (int kc = k0; kc < k1; ++kc, ++c, at.next(p.stages)) {
                    uint64_t * bar = full + at.s;
                    if (at.round != 0) {
                        ok = gmm_wait_one<CTAS>(empty + at.s, (at.round - 1u) & 1u, &abort_flag);
                        if (!ok) break;
                        ++done;
                    }
                    uint8_t * st = ring + (uint32_t)at.s * stage_bytes;
                    if (rank == 0) mbar_arrive_expect_tx(bar, bytes);
                    gmm_tma_3d<CTAS>(st, &p.wmap, kc * kGmmK, m0, q.g, bar);
                    if (MODE != GMM_PLAIN) gmm_tma_3d<CTAS>(st + kABytes / 2, &p.umap, kc * kGmmK, m0, q.g, bar);
                    for (int b = 0; b < boxes; ++b)
                        gmm_tma_2d<CTAS>(st + kABytes + (uint32_t)b * (p.box * 128u), &p.xmap, kc * kGmmK, r0 + b * p.box, bar);
                }
            }
            // (the issuer's commits arrive in both CTAs of a pair: the last ones too, before either leaves)
            for (int i = max(0, c - p.stages); i < c && ok; ++i)
                ok = gmm_wait_one<CTAS>(empty + i % p.stages, (uint32_t)((i / p.stages) & 1), &abort_flag);
            if (!ok && rank == 0) {
                // copies in flight land before the CTA leaves
                volatile int none = 0;
                for (int i = done; i < c; ++i) gmm_wait_one<CTAS>(full + i % p.stages, (uint32_t)((i / p.stages) & 1), &none);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------ MMA issuer
        if (rank == 0 && elect_one()) {
            int it = 0;
            RingPos at;
            bool ok = true;
            const uint64_t da0 = umma_desc_sw128(ring, 1024u), db0 = umma_desc_sw128(ring + kABytes, 1024u);
            for (Work w = start(); w.t < tiles && ok; advance(w)) {
                const GmmTile q = gmm_tile<kRound, SRC>(p, pre, w.t, kOut * CTAS);
                const int k0 = first_chunk(w), k1 = end_chunk(w);
                const uint32_t n = (uint32_t)((q.cnt + kRound - 1) / kRound * kRound);
                const uint32_t idesc = umma_idesc_f16(p.bf16 != 0, kGmmRows * CTAS, n);
                for (int kc = k0; kc < k1 && ok; ++it) {
                    const int b = it % kBufs, end = p.seg ? min(kc + p.seg, k1) : k1;
                    if (it >= kBufs) ok = gmm_wait_one<CTAS>(acc_empty + b, (uint32_t)((it / kBufs - 1) & 1), &abort_flag);
                    const uint32_t d = tbase + (uint32_t)(b * p.acc);
                    uint32_t more = 0;                                   // the first MMA overwrites the accumulator
                    for (; kc < end && ok; ++kc, at.next(p.stages)) {
                        ok = gmm_wait_one<CTAS>(full + at.s, at.round & 1u, &abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        // (a stage's address only touches the low word: 14 bits of 16 bytes)
                        const uint64_t off = (uint64_t)(((uint32_t)at.s * stage_bytes) >> 4);
#pragma unroll
                        for (int i = 0; i < kGmmK / 16; ++i)
                            mma_f16<CTAS>(d, da0 + off + (uint64_t)(2 * i), db0 + off + (uint64_t)(2 * i), idesc, more | (uint32_t)i);
                        if constexpr (MODE == GMM_DUAL) {
#pragma unroll
                            for (int i = 0; i < kGmmK / 16; ++i)
                                mma_f16<CTAS>(d + 256u, da0 + (kGmmATile >> 4) + off + (uint64_t)(2 * i), db0 + off + (uint64_t)(2 * i),
                                              idesc, more | (uint32_t)i);
                        }
                        if constexpr (SRC != GMM_TILES) {
                            for (int part = 1; part < p.parts; ++part)
#pragma unroll
                                for (int i = 0; i < kGmmK / 16; ++i)
                                    mma_f16<CTAS>(d, da0 + (uint64_t)part * (kGmmATile >> 4) + off + (uint64_t)(2 * i),
                                                  db0 + off + (uint64_t)(2 * i), idesc, 1u);
                        }
                        more = 1;
                        gmm_commit<CTAS>(empty + at.s);
                    }
                    if (ok) gmm_commit<CTAS>(acc_full + b);
                }
            }
            // MMAs in flight end before TMEM is freed and the CTA leaves, whoever gave up: where this
            // thread did not, the last chunk's commit says so
            volatile int none = 0;
            if (!ok) {
                gmm_commit<CTAS>(&drained);
                gmm_wait_one<CTAS>(&drained, 0, &none);
            } else if (it > 0) {
                const bool wrap = at.s == 0;
                gmm_wait_one<CTAS>(empty + (wrap ? p.stages : at.s) - 1, (at.round - (wrap ? 1u : 0u)) & 1u, &none);
            }
        }
        __syncwarp();
    } else if (warp < 2 + kGather) {
        // -------------------------------------------------- gathered rows
        // four rows of 128 bytes per copy (tile::gather4), up to 32 rows per
        // warp: the warp looks its rows up, one thread issues the copies. A
        // warp without rows in a tile still copies four: a stage that does not
        // wait for it could go round the ring twice before it looks, and the
        // parity of its barrier would then say the opposite.
        const int gw = warp - 2;
        if (gw < gathering) {
            int32_t * rows = gather_rows + gw * 32;
            RingPos at;
            bool ok = true;
            for (Work w = start(); w.t < tiles && ok; advance(w)) {
                const GmmTile q = gmm_tile<kRound, SRC>(p, pre, w.t, kOut * CTAS);
                const int k0 = first_chunk(w), k1 = end_chunk(w);
                const int half = ((q.cnt + kRound - 1) / kRound * kRound) / CTAS;
                const int n = max(0, min(half, q.cnt - rank * half));             // this CTA's rows
                const int quads = gather_quads(n, gw);
                // (rows behind the last repeat it)
                const int o = p.order[q.row0 + min(rank * half + min(gw * 32 + lane, max(n - 1, 0)), q.cnt - 1)];
                int row = o / p.gather;
                if (o < 0 || row >= p.x_rows) {
                    record_error(GX_DEVERR_DOMAIN);
                    row = 0;
                }
                __syncwarp();
                rows[lane] = row;
                __syncwarp();
                if (elect_one()) {
                    int4 of[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) of[i] = *reinterpret_cast<const int4 *>(rows + i * 4);
                    RingPos on = at;
                    for (int kc = k0; kc < k1; ++kc, on.next(p.stages)) {
                        if (on.round != 0) {
                            ok = gmm_wait_one<CTAS>(empty + on.s, (on.round - 1u) & 1u, &abort_flag);
                            if (!ok) break;
                        }
                        uint8_t * to = ring + (uint32_t)on.s * stage_bytes + kABytes + (uint32_t)gw * 4096u;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (i < quads)
                                gmm_gather4<CTAS>(to + i * 512, &p.xmap, kc * kGmmK, of[i].x, of[i].y, of[i].z, of[i].w, full + on.s);
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                at.skip(k1 - k0, p.stages);
            }
        }
    } else if (SRC != GMM_TILES && warp >= 2 + kGather + kEpi) {
        // --------------------------------- tiles of weights from their blocks
        // Four warps a tile of 128 rows, a lane a row, the two fours taking the
        // chunks of 64 elements in turn (a stage's barrier is at most one phase
        // behind what they wait for: they have waited for the chunk two before, in
        // another stage, and stages come free in order). The rows' pieces come into a
        // ring that two warps share: by TMA boxes, or, where rows do not start on
        // 16 bytes, by bulk copies, a lane a row (32 of those keep a warp for 2800
        // cycles; cp.async would be waited for by every fence that shows a tile to
        // the tensor cores).
        if constexpr (SRC != GMM_TILES) {
            constexpr bool Q41 = SRC >= GMM_Q4_1_F16, BF = SRC == GMM_Q4_0_BF16 || SRC == GMM_Q4_1_BF16;
            constexpr int kPair = Q41 ? 40 : 36, kWords = kPair / 4;
            constexpr uint32_t kPitch = gmm_q4_pitch(Q41);
            const int qw = warp - (2 + kGather + kEpi), rg = qw & 3, odd = qw >> 2;
            uint8_t * my = raw + (uint32_t)rg * (kGmmQ4Stages * 32u * kPitch) + (uint32_t)lane * kPitch;
            const uint8_t * w_of = GLU && rg >= 2 ? p.w1 : p.w0;
            const uint8_t * const w_end = w_of + (int64_t)(p.G - 1) * p.nb02 + (int64_t)(p.N - 1) * p.nb01 + (int64_t)nk * kPair;
            const int base_row = (GLU ? (rg & 1) * 32 : rg * 32) + lane;
            const int steps = (nk + kGmmQ4Chunks - 1) / kGmmQ4Chunks;        // stages of a tile
            bool ok = true;
            // the copies run a stage or two ahead (the first four's)
            Work aw = start();
            GmmTile aq{};
            int a_step = 0, issued = 0;
            if (aw.t < tiles) aq = gmm_tile<kRound, SRC>(p, pre, aw.t, kOut * CTAS);
            auto step_on = [&] {
                ++issued;
                if (++a_step == steps) {
                    a_step = 0;
                    advance(aw);
                    if (aw.t < tiles) aq = gmm_tile<kRound, SRC>(p, pre, aw.t, kOut * CTAS);
                }
            };
            auto fetch = [&] {
                if (odd != 0 || aw.t >= tiles || !ok) return;
                const int s = issued % kGmmQ4Stages;
                if (issued >= kGmmQ4Stages) ok = gmm_wait<1>(&raw_empty[rg][s], (uint32_t)((issued / kGmmQ4Stages - 1) & 1), &abort_flag);
                if (!ok) return;
                if (p.boxes) {
                    // (one copy; words behind the row's and rows behind the last are zeros)
                    if (elect_one()) {
                        mbar_arrive_expect_tx(&raw_full[rg][s], 32u * kPitch);
                        tma_load_3d(raw + (uint32_t)(rg * kGmmQ4Stages + s) * (32u * kPitch), GLU && rg >= 2 ? &p.umap : &p.wmap,
                                    a_step * (kGmmQ4Chunks * kWords), aq.m0 + rank * kOut + base_row - lane, aq.g, &raw_full[rg][s]);
                    }
                    __syncwarp();
                    step_on();
                    return;
                }
                const int m = aq.m0 + rank * kOut + base_row, n = min(kGmmQ4Chunks, nk - a_step * kGmmQ4Chunks);
                const uint8_t * a = w_of + (int64_t)aq.g * p.nb02 + (int64_t)m * p.nb01 + (int64_t)a_step * (kGmmQ4Chunks * kPair);
                const uint32_t skew = (uint32_t)reinterpret_cast<uintptr_t>(a) & 15u;
                uint32_t bytes = m < p.N ? (skew + (uint32_t)(n * kPair) + 15u) & ~15u : 0u;     // (rows behind the last: nothing)
                const uint8_t * from = a - skew;
                uint8_t * to = my + (uint32_t)s * (32u * kPitch);
                // (the last row's last piece ends with the matrix: what is not whole 16 bytes is moved by hand)
                if (bytes != 0u && from + bytes > w_end) {
                    bytes -= 16u;
                    for (const uint8_t * b = from + bytes; b < w_end; b += 4)
                        *reinterpret_cast<uint32_t *>(to + (b - from)) = *reinterpret_cast<const uint32_t *>(b);
                }
                const uint32_t sum = __reduce_add_sync(0xffffffffu, bytes);
                __syncwarp();                            // (that lane's stores, before the arrival that shows them to the other four's warp)
                if (lane == 0) mbar_arrive_expect_tx(&raw_full[rg][s], sum);
                __syncwarp();
                if (bytes != 0u) bulk_g2s(to, from, bytes, &raw_full[rg][s]);
                step_on();
            };
            fetch();
            const int row = rg * 32 + lane;
            RingPos at;
            int taken = 0, lead = odd;                  // lead: chunks of others before the next own one
            if (odd) at.next(p.stages);
            for (Work w = start(); w.t < tiles && ok; advance(w)) {
                const GmmTile q = gmm_tile<kRound, SRC>(p, pre, w.t, kOut * CTAS);
                // where the lane's row starts inside its 16 bytes
                const uint32_t low = (uint32_t)reinterpret_cast<uintptr_t>(w_of) + (uint32_t)q.g * (uint32_t)p.nb02 +
                                     (uint32_t)(q.m0 + rank * kOut + base_row) * (uint32_t)p.nb01;
                for (int kc = 0; kc < nk && ok; kc += kGmmQ4Chunks) {
                    const int rs = taken % kGmmQ4Stages, n = min(kGmmQ4Chunks, nk - kc);
                    fetch();
                    ok = ok && gmm_wait<1>(&raw_full[rg][rs], (uint32_t)((taken / kGmmQ4Stages) & 1), &abort_flag);
                    if (!ok) break;
                    const uint32_t skew = (low + (uint32_t)(kc * kPair)) & 15u;
                    const uint32_t src = smem_u32(my + (uint32_t)rs * (32u * kPitch));
                    int in = lead;
                    for (; in < n; in += 2) {
                        // the chunk's words, out of three or four pieces of 16 bytes
                        constexpr int kPieces = (kPair + 12 + 15) / 16;
                        uint32_t v[4 * kPieces];
                        const uint32_t o = skew + (uint32_t)(in * kPair), a = src + (o & ~15u);
#pragma unroll
                        for (int i = 0; i < kPieces; ++i)
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(v[4 * i]), "=r"(v[4 * i + 1]), "=r"(v[4 * i + 2]), "=r"(v[4 * i + 3])
                                         : "r"(a + 16u * (uint32_t)i)
                                         : "memory");
#pragma unroll
                        for (int i = 0; i + 2 < 4 * kPieces && i < kWords + 1; ++i) v[i] = o & 8u ? v[i + 2] : v[i];
#pragma unroll
                        for (int i = 0; i < kWords; ++i) v[i] = o & 4u ? v[i + 1] : v[i];
                        const uint32_t tile = smem_u32(ring + (uint32_t)at.s * stage_bytes) + (uint32_t)row * 128u;
                        auto place = [&](int blk, int i) { return tile + (uint32_t)(((4 * blk + i) ^ (row & 7)) << 4); };
                        auto mine = [&] { return at.round == 0 || gmm_wait<CTAS>(empty + at.s, (at.round - 1u) & 1u, &abort_flag); };
                        if constexpr (Q41) {
                            ok = mine();
                            if (!ok) break;
#pragma unroll
                            for (int blk = 0; blk < 2; ++blk) {
                                const float2 head = __half22float2(*reinterpret_cast<const __half2 *>(&v[5 * blk]));
                                const float d = head.x, c = __fmaf_rn(-16.0f, d, head.y);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    // elements 8 i .. 8 i + 7 of the block: d q + m
                                    float f[8];
#pragma unroll
                                    for (int j = 0; j < 2; ++j) {
                                        const uint32_t b = v[5 * blk + 1 + 2 * (i & 1) + j];
                                        q4_spread(((i < 2 ? b << 3 : b >> 1) & 0x78787878u) | 0x80808080u, f + 4 * j);
                                    }
#pragma unroll
                                    for (int j = 0; j < 8; ++j) f[j] = __fmaf_rn(f[j], d, c);
                                    q4_put<BF>(f, place(blk, i), p.parts);
                                }
                            }
                        } else {
                            // words 0 .. 4 and 4 .. 8: the first block's codes begin in the middle of a word
#pragma unroll
                            for (int blk = 0; blk < 2; ++blk) {
                                const __half2 head = *reinterpret_cast<const __half2 *>(&v[4 * blk]);
                                const Q4Scale<BF> d(blk == 0 ? __low2half(head) : __high2half(head));
                                uint32_t qs[4], q[4][4], t[4][4], w[4][4];
#pragma unroll
                                for (int i = 0; i < 4; ++i) qs[i] = blk == 0 ? __byte_perm(v[i], v[i + 1], 0x5432) : v[5 + i];
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    // elements 8 i .. 8 i + 7 of the block
                                    q4_pairs<BF>(qs[2 * (i & 1)], i >= 2, q[i][0], q[i][1]);
                                    q4_pairs<BF>(qs[2 * (i & 1) + 1], i >= 2, q[i][2], q[i][3]);
#pragma unroll
                                    for (int j = 0; j < 4; ++j) w[i][j] = q4_first_part<BF>(q[i][j], t[i][j], d);
                                }
                                // (the first half is made before the stage is free)
                                if (blk == 0) ok = mine();
                                if (!ok) break;
#pragma unroll
                                for (int i = 0; i < 4; ++i) q4_store(place(blk, i), w[i]);
                                if (p.parts > 1) {
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
#pragma unroll
                                        for (int j = 0; j < 4; ++j) w[i][j] = q4_second_part<BF>(w[i][j], q[i][j], t[i][j], d);
                                        q4_store(place(blk, i) + kGmmATile, w[i]);
                                    }
                                }
                            }
                            if (!ok) break;
                        }
                        fence_async_smem();
                        __syncwarp();
                        // (the fence has put the tile where the tensor cores of both CTAs see it: no release over the cluster)
                        if (lane == 0) gmm_arrive<CTAS>(full + at.s);
                        at.next(p.stages);
                        at.next(p.stages);
                    }
                    lead = in - n;
                    __syncwarp();
                    if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&raw_empty[rg][rs])) : "memory");
                    ++taken;
                }
            }
            // copies in flight land before the CTA leaves
            volatile int none = 0;
            for (int i = 0; i < kGmmQ4Stages && !ok; ++i)
                if (issued > i) gmm_wait<1>(&raw_full[rg][i], (uint32_t)((issued - 1 - i) / kGmmQ4Stages & 1), &none);
        }
    } else {
        // -------------------------------------------------------- epilogue
        const int quad = warp & 3;             // TMEM lanes 32 * quad ..
        const int ew = warp - 2 - kGather;
        uint8_t * stage = staging + (uint32_t)ew * (kGmmStaging / kEpi);
        const bool vec = ((reinterpret_cast<uintptr_t>(p.dst) | (uintptr_t)p.nbd1) & 15u) == 0;
        const uint32_t lanes = (uint32_t)quad << 21, dsum = tbase + lanes + 2u * (uint32_t)p.acc;
        int it = 0, xb = 0, i_tile = 0;
        bool ok = true;
        Work w = start();
        for (; w.t < tiles && ok; advance(w)) {
            const GmmTile q = gmm_tile<kRound, SRC>(p, pre, w.t, kOut * CTAS);
            const int k0 = first_chunk(w), k1 = end_chunk(w);
            const int nseg = p.seg ? (k1 - k0 + p.seg - 1) / p.seg : 1;
            // the order of the first columns' rows is on its way before the sums are there
            const bool ordered = p.gather != 0 || p.scatter != 0;
            const int col0 = 32 * (ew / 4);
            int o_next = ordered && col0 + lane < q.cnt ? p.order[q.row0 + col0 + lane] : 0;
            uint32_t d = 0;
            for (int sg = 0; sg < nseg && ok; ++sg, ++it) {
                const int b = it % kBufs;
                ok = gmm_wait<CTAS>(acc_full + b, (uint32_t)((it / kBufs) & 1), &abort_flag);
                if (!ok) break;
                tc_fence_after();
                d = tbase + lanes + (uint32_t)(b * p.acc);
                if (sg + 1 == nseg) break;
                // an earlier segment of K: onto the running sums in TMEM, rounded to nearest
                for (int c0 = 0; c0 < q.cnt; c0 += 32) {
                    uint32_t v[32];
                    tmem_ld32(d + (uint32_t)c0, v);
                    if (sg > 0) {
                        uint32_t w[32];
                        tmem_ld32(dsum + (uint32_t)c0, w);
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__fadd_rn(__uint_as_float(w[i]), __uint_as_float(v[i])));
                    }
                    tmem_st32(dsum + (uint32_t)c0, v);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) gmm_arrive<CTAS>(acc_empty + b);
            }
            if constexpr (GLU) ok = pair_agrees(1 + (quad & 1), ok);
            if (!ok) break;
            // the tile's f32 sums of columns c0 .. c0 + 31
            auto sums = [&](int c0, uint32_t (&v)[32]) {
                tmem_ld32(d + (uint32_t)c0, v);
                if (nseg > 1) {
                    uint32_t w[32];
                    tmem_ld32(dsum + (uint32_t)c0, w);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__fadd_rn(__uint_as_float(w[i]), __uint_as_float(v[i])));
                }
            };
            const int leader = i_tile % split, pb = i_tile & 1;
            if (w.shared) {
                // K is shared: the partial sums go to shared memory, and the
                // tile's leader (in turn) adds them up in CTA order
                if (i_tile >= 2) ok = gmm_wait<2>(part_free + pb, (uint32_t)((i_tile / 2 - 1) & 1), &abort_flag);
                if (ok) {
                    uint32_t v[32];
                    sums(0, v);
                    float * to = part + (pb * p.nt) * kGmmRows + quad * 32 + lane;
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (i < q.cnt) to[i * kGmmRows] = __uint_as_float(v[i]);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        gmm_arrive<CTAS>(acc_empty + it % kBufs);
                        arrive_at(&part_full, leader);
                    }
                    if (me == leader) ok = gmm_wait<2>(&part_full, (uint32_t)((i_tile / split) & 1), &abort_flag);
                }
                if constexpr (GLU) ok = pair_agrees(1 + (quad & 1), ok);
                if (!ok) break;
                ++i_tile;
                if (me != leader) {
                    ++it;
                    continue;
                }
            }
            const int n0 = q.m0 + rank * kOut + (GLU ? quad & 1 : quad) * 32;
            constexpr int kStep = 8 * kEpi;              // (dual: two warps of four share the columns)
            for (int c0 = col0; c0 < q.cnt; c0 += kStep) {
                const int o = o_next;
                o_next = ordered && c0 + kStep + lane < q.cnt ? p.order[q.row0 + c0 + kStep + lane] : 0;
                uint32_t v[32], u[MODE == GMM_DUAL ? 32 : 1];
                if (w.shared) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0u;
                    for (int c = 0; c < split; ++c) {
                        const uint32_t from = peer_addr(part + (pb * p.nt) * kGmmRows + quad * 32 + lane, c);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i < q.cnt)
                                v[i] = __float_as_uint(__fadd_rn(__uint_as_float(v[i]), ld_peer(from + (uint32_t)i * (kGmmRows * 4u))));
                    }
                } else if constexpr (MODE == GMM_DUAL) {
                    tmem_ld32_start(d + (uint32_t)c0, v);
                } else {
                    sums(c0, v);
                }
                if constexpr (MODE == GMM_DUAL) {
                    tmem_ld32_start(d + 256u + (uint32_t)c0, u);
                    tmem_ld32_end(v);
                    tmem_ld32_end(u);
                }
                // after its last columns are read a warp gives the accumulator back, and then finishes them
                if (!w.shared && c0 + kStep >= q.cnt) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) gmm_arrive<CTAS>(acc_empty + it % kBufs);
                }
                bool nan = false;
                int my = c0 + lane < q.cnt ? gmm_dst_row(p, q.row0 + c0 + lane, o, nan) : -1;
                const unsigned nans = __ballot_sync(0xffffffffu, nan);
                if constexpr (GLU) {
                    // quads 0, 1 hold gate rows, quads 2, 3 the same up rows:
                    // each of a pair finishes 16 of the 32 columns
                    const int pair = quad & 1, up = quad >> 1;
                    float * sendp = xchg + (((xb * 2 + pair) * 2 + up) * 16) * 32 + lane;
                    const float * recvp = xchg + (((xb * 2 + pair) * 2 + (up ^ 1)) * 16) * 32 + lane;
                    float own[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        sendp[i * 32] = __uint_as_float(up ? v[i] : v[16 + i]);
                        own[i] = __uint_as_float(up ? v[16 + i] : v[i]);
                    }
                    asm volatile("bar.sync %0, 64;" ::"r"(1 + pair) : "memory");
                    my = __shfl_sync(0xffffffffu, my, (lane & 15) + 16 * up);
                    float gv[16], uv[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float other = recvp[i * 32];
                        gv[i] = up ? other : own[i];
                        uv[i] = up ? own[i] : other;
                    }
                    gmm_act_all<16>(p, gv, uv);
#pragma unroll
                    for (int i = 0; i < 16; ++i) own[i] = (nans >> (i + 16 * up)) & 1u ? kNan : gv[i];
                    xb ^= 1;
                    put_rows_as<16>(p, stage, own, my, n0, vec);
                } else if constexpr (MODE == GMM_DUAL) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float own[16], uv[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            own[i] = __uint_as_float(v[16 * half + i]);
                            uv[i] = __uint_as_float(u[16 * half + i]);
                        }
                        gmm_act_all<16>(p, own, uv);
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if ((nans >> (i + 16 * half)) & 1u) own[i] = kNan;
                        put_rows_as<16>(p, stage, own, __shfl_sync(0xffffffffu, my, (lane & 15) + 16 * half), n0, vec);
                    }
                } else {
                    float own[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) own[i] = (nans >> i) & 1u ? kNan : __uint_as_float(v[i]);
                    put_rows_as<32>(p, stage, own, my, n0, vec);
                }
            }
            if (w.shared) {
                __syncwarp();
                arrive_all(part_free + pb, split);
            } else if (col0 >= q.cnt) {
                // (a warp without columns in this tile)
                tc_fence_before();
                __syncwarp();
                if (lane == 0) gmm_arrive<CTAS>(acc_empty + it % kBufs);
            }
            ++it;
        }
        if constexpr (SRC != GMM_TILES) {
            if (!ok) gmm_fill_nan<kRound, SRC>(p, pre, w.t, units, tiles, kOut * CTAS, rank * kOut + (GLU ? quad & 1 : quad) * 32);
        }
    }
    tc_fence_before();
    if (CTAS * split == 1) __syncthreads(); else cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        gmm_tmem_free<CTAS>(tbase, 512);
    }
}

}  // namespace gx
