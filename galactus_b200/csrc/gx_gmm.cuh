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
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gx_grouped_plan.h"
#include "gx_tc.cuh"

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
};

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

// and of a value over the two warps that share a named barrier
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
template <int ROUND>
__device__ __forceinline__ GmmTile gmm_tile(const GmmParams & p, const int32_t * pre, int t, int rows) {
    GmmTile r;
    const int tt = t / p.mt;
    r.m0 = (t - tt * p.mt) * rows;
    r.g = tile_group(pre, p.G, tt);
    const int lo = p.offsets[r.g], hi = p.offsets[r.g + 1];
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
__device__ __forceinline__ int gmm_dst_row(const GmmParams & p, int j, int o, bool & nan) {
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
template <bool OAI, bool FAST>
__device__ __forceinline__ float gmm_act(const GmmParams & p, float g, float u) {
    if (!OAI) return __fmul_rn(gmm_sigmoid_times<FAST>(g, -g), u);
    const float x = p.limit < g ? p.limit : g;
    const float y = u < -p.limit ? -p.limit : (p.limit < u ? p.limit : u);
    return __fmul_rn(gmm_sigmoid_times<FAST>(x, __fmul_rn(p.alpha, -x)), __fadd_rn(y, 1.0f));
}
// of N values at once: g becomes the result (the choices stay outside the
// loop, so that the values' chains of operations overlap)
template <bool OAI, bool FAST, int N>
__device__ __forceinline__ void gmm_act_each(const GmmParams & p, float (&g)[N], const float (&u)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = gmm_act<OAI, FAST>(p, g[i], u[i]);
}
template <int N>
__device__ __forceinline__ void gmm_act_all(const GmmParams & p, float (&g)[N], const float (&u)[N]) {
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

template <int CTAS, int MODE>
__global__ void __launch_bounds__(gmm_threads(MODE), 1) k_gmm(const __grid_constant__ GmmParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[kGmmMaxStages], empty[kGmmMaxStages], acc_full[2], acc_empty[2], part_full, part_free[2], drained;
    __shared__ uint32_t tslot;
    __shared__ int4 gather_mem[kGmmGatherWarps * 8];
    __shared__ int32_t wsum[gmm_threads(MODE) / 32];
    __shared__ int abort_flag;
    int32_t * gather_rows = reinterpret_cast<int32_t *>(gather_mem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = CTAS == 1 ? 0 : (int)(blockIdx.x & 1);              // CTA of the pair; 0 leads
    const int split = CTAS == 1 ? p.split : 1;
    const int me = CTAS == 1 ? (int)blockIdx.x % split : 0;             // share of K
    constexpr bool GLU = MODE == GMM_GLU;
    constexpr int kBufs = MODE == GMM_DUAL ? 1 : 2;                      // accumulators that take turns
    constexpr int kEpi = gmm_epi_warps(MODE);
    constexpr uint32_t kABytes = gmm_a_bytes(MODE);
    uint8_t * ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t stage_bytes = gmm_stage_bytes(CTAS, p.nt, MODE);
    uint8_t * staging = ring + (uint32_t)p.stages * stage_bytes;
    float * xchg = reinterpret_cast<float *>(staging + kGmmStaging);
    float * part = xchg + (GLU ? kGmmXchg / 4 : 0u);                     // [2][nt][128] partial sums of a shared tile
    int32_t * pre = reinterpret_cast<int32_t *>(part + (split > 1 ? 2 * p.nt * kGmmRows : 0));
    constexpr int kOut = gmm_out_rows(MODE);                             // result rows of a CTA's tile
    constexpr int kRound = 16 * CTAS;                                    // MMA N: a multiple of this

    if (tid == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + i, 1);
            mbar_init(acc_empty + i, kEpi * CTAS);
        }
        mbar_init(&part_full, (uint32_t)(kEpi * split));
        for (int i = 0; i < 2; ++i) mbar_init(part_free + i, kEpi);
        mbar_init(&drained, 1);
        abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) gmm_tmem_alloc<CTAS>(&tslot, 512);
    tile_prefix(pre, wsum, p.G, p.nt, p.most, [&](int g) { return group_rows_of(p.offsets, g, p.n_rows); });
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

    if (warp == 0) {
        // ------------------------------------------- weights, rows in place
        if (elect_one()) {
            int c = 0, done = 0;       // chunks started; chunks whose stage was handed back
            RingPos at;
            bool ok = true;
            for (Work w = start(); w.t < tiles && ok; advance(w)) {
                const GmmTile q = gmm_tile<kRound>(p, pre, w.t, kOut * CTAS);
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
                const GmmTile q = gmm_tile<kRound>(p, pre, w.t, kOut * CTAS);
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
                        more = 1;
                        gmm_commit<CTAS>(empty + at.s);
                    }
                    if (ok) gmm_commit<CTAS>(acc_full + b);
                }
            }
            if (!ok) {
                volatile int none = 0;
                gmm_commit<CTAS>(&drained);
                gmm_wait_one<CTAS>(&drained, 0, &none);
            }
        }
        __syncwarp();
    } else if (warp < 2 + kGmmGatherWarps) {
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
                const GmmTile q = gmm_tile<kRound>(p, pre, w.t, kOut * CTAS);
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
    } else {
        // -------------------------------------------------------- epilogue
        const int quad = warp & 3;             // TMEM lanes 32 * quad ..
        const int ew = warp - 2 - kGmmGatherWarps;
        uint8_t * stage = staging + (uint32_t)ew * (kGmmStaging / kEpi);
        const bool vec = ((reinterpret_cast<uintptr_t>(p.dst) | (uintptr_t)p.nbd1) & 15u) == 0;
        const uint32_t lanes = (uint32_t)quad << 21, dsum = tbase + lanes + 2u * (uint32_t)p.acc;
        int it = 0, xb = 0, i_tile = 0;
        bool ok = true;
        for (Work w = start(); w.t < tiles && ok; advance(w)) {
            const GmmTile q = gmm_tile<kRound>(p, pre, w.t, kOut * CTAS);
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
    }
    tc_fence_before();
    if (CTAS * split == 1) __syncthreads(); else cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        gmm_tmem_free<CTAS>(tbase, 512);
    }
}

}  // namespace gx
