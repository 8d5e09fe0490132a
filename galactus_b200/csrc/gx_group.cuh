// Rows of a micro-batch grouped by expert, by adapter, or by adapter and
// expert (sm_100a): a stable counting sort of the P = k*T (token, slot) pairs.
//
//   key(p)   = adapter[t] * n_as + ids[t, s]   (either part may be absent)
//   order    the pairs by ascending key, pairs of one key by ascending p;
//            pairs of no group (a negative id or adapter) come last
//   offsets  where each group starts; offsets[G] = the pairs that have one
//
// ONE launch: the pairs are cut into contiguous segments, one per warp, over
// a cluster of up to 8 CTAs. Every warp counts its segment's keys into a
// histogram of its own, the counts become starting positions by a prefix over
// warps, over the CTAs of the cluster (read from their shared memory) and
// over the groups, and a second pass over the same pairs writes them out
// (match.any ranks a step's equal keys by lane: nothing depends on timing).
// The number of counting warps follows the group count: their histograms must
// fit in shared memory.
//
// Bound by latency (a 2048-token batch is 131 KB of indices, 20 ns of
// bandwidth): the design keeps the dependent steps few and the launch single.
// On a B200: 3.1 us for 8 pairs, 7.2 us for 16384 pairs in 128 groups, 10 us
// for 4136 pairs in 1536 groups; 16384 pairs take 22 us in one CTA.
#pragma once

#include <cooperative_groups.h>

#include "gx_device.cuh"

namespace gx {

constexpr int kGroupMaxGroups = 8192;
constexpr int kGroupCluster = 8;
constexpr uint32_t kGroupSmem = 200u * 1024u;

struct GroupParams {
    const int32_t * ids;      // [T, k], nbi1 bytes between tokens, or NULL (k = 1)
    int64_t nbi1;
    const int32_t * adapter;  // [T] or NULL
    int32_t k, n_as, n_adapters, G;
    int32_t P;
    uint32_t div_m, div_l;    // t = q / k as (umulhi(q, div_m) + q) >> div_l
    int32_t warps;            // counting warps per CTA
    int32_t seg;              // pairs per counting warp, a multiple of 32
    int32_t * order;
    int32_t * offsets;
};

// group of pair q, G for none
__device__ __forceinline__ int group_key(const GroupParams & p, int q) {
    const int t = (int)((__umulhi((uint32_t)q, p.div_m) + (uint32_t)q) >> p.div_l), s = q - t * p.k;
    int key = 0;
    bool bad = false;
    if (p.ids != nullptr) {
        key = *reinterpret_cast<const int32_t *>(reinterpret_cast<const char *>(p.ids) + (int64_t)t * p.nbi1 + 4ll * s);
        bad = key >= p.n_as;
    }
    if (p.adapter != nullptr) {
        const int a = p.adapter[t];
        bad = bad || a >= p.n_adapters;
        key = (a < 0 || key < 0) ? -1 : bad ? -1 : a * p.n_as + key;
    }
    if (bad) record_error(GX_DEVERR_DOMAIN);
    return (bad || key < 0) ? p.G : key;
}

__global__ void __launch_bounds__(1024) k_group_rows(const __grid_constant__ GroupParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ int32_t gsm[];
    const int G1 = p.G + 1;
    int32_t * total = gsm;             // [G1] pairs of each group in this CTA
    int32_t * base = total + G1;       // [G1] first position of this CTA's pairs of the group
    int32_t * hist = base + G1;        // [warps][G1]
    __shared__ int32_t wsum[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nt = blockDim.x;
    const cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), ncta = (int)cl.num_blocks();

    for (int i = tid; i < p.warps * G1; i += nt) hist[i] = 0;
    __syncthreads();
    const int64_t s0 = ((int64_t)rank * p.warps + warp) * p.seg;
    const int first = (int)(s0 < p.P ? s0 : p.P);
    const int last = (int)(s0 + p.seg < p.P ? s0 + p.seg : p.P);
    int32_t * mine = hist + warp * G1;
    if (warp < p.warps) {
        int ahead = first + lane < last ? group_key(p, first + lane) : G1;
        for (int q0 = first; q0 < last; q0 += 32) {
            const int key = ahead;
            ahead = q0 + 32 + lane < last ? group_key(p, q0 + 32 + lane) : G1;
            if (key < G1) atomicAdd(mine + key, 1);            // (a count: the order of the adds does not show)
        }
    }
    __syncthreads();
    // per group: exclusive prefix over this CTA's warps, and the CTA's total
    for (int g = tid; g < G1; g += nt) {
        int run = 0;
        for (int w = 0; w < p.warps; ++w) {
            const int c = hist[w * G1 + g];
            hist[w * G1 + g] = run;
            run += c;
        }
        total[g] = run;
    }
    if (ncta > 1) cl.sync(); else __syncthreads();
    // each thread takes a run of consecutive groups: their totals over the
    // cluster, scanned over the block, are the group borders
    const int per = (G1 + nt - 1) / nt;
    const int g0 = min(tid * per, G1), g1 = min(g0 + per, G1);
    int sum = 0;
    for (int g = g0; g < g1; ++g) {
        int all = 0, before = 0;
        for (int c = 0; c < ncta; ++c) {
            const int v = ncta > 1 ? *cl.map_shared_rank(total + g, c) : total[g];
            if (c < rank) before += v;
            all += v;
        }
        base[g] = sum + before;
        sum += all;
    }
    int inc = sum;
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int pre = inc - sum;
    for (int w = 0; w < warp; ++w) pre += wsum[w];
    for (int g = g0; g < g1; ++g) {
        base[g] += pre;
        if (rank == 0) p.offsets[g] = base[g];   // nothing stands before rank 0's pairs of a group
    }
    // (the sync also keeps every CTA's totals alive until all have read them)
    if (ncta > 1) cl.sync(); else __syncthreads();
    if (warp < p.warps) {
        int ahead = first + lane < last ? group_key(p, first + lane) : G1;
        for (int q0 = first; q0 < last; q0 += 32) {
            const int q = q0 + lane, key = ahead;
            ahead = q + 32 < last ? group_key(p, q + 32) : G1;
            const unsigned peers = __match_any_sync(0xffffffffu, key);
            const int at = __popc(peers & ((1u << lane) - 1u));
            if (key < G1) p.order[base[key] + mine[key] + at] = q;
            __syncwarp();
            if (key < G1 && at == 0) mine[key] += __popc(peers);
            __syncwarp();
        }
    }
}

}  // namespace gx
