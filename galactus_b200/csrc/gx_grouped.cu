// Entry points of the operators on grouped rows: the grouping, the products
// with unquantised experts and the adapters' low-rank deltas. No C++
// exception crosses this boundary; every entry point returns GX_*.
#include <algorithm>

#include "gx_group.cuh"
#include "gx_kernels.h"
#include "gx_launch.h"
#include "gx_lora.cuh"

namespace gx {

cudaError_t read_and_clear_grouped_error(int * code) {
    int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(code, g_dev_error, sizeof(int));
    if (e != cudaSuccess) return e;
    return cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(int));
}

namespace {

// One CTA per row and 1024 elements, four elements a thread (more in rows of
// over 65535 x 1024).
__global__ void __launch_bounds__(256) k_round_rows(bool bf16, const float * src, int ne0, int64_t nb1, uint8_t * dst,
                                                    int64_t stride) {
    const float * s = reinterpret_cast<const float *>(reinterpret_cast<const uint8_t *>(src) + (int64_t)blockIdx.x * nb1);
    uint8_t * d = dst + (int64_t)blockIdx.x * stride;
    for (int64_t c = (int64_t)blockIdx.y * 1024; c < ne0; c += (int64_t)gridDim.y * 1024)
        for (int64_t i = c + threadIdx.x; i < ne0 && i < c + 1024; i += 256) store_out(d, (int)i, s[i], bf16 ? GMM_BF16 : GMM_F16);
}

}  // namespace

cudaError_t launch_round_rows(bool bf16, const float * src, int64_t ne0, int64_t nrows, int64_t nb1, uint8_t * dst,
                              int64_t stride, cudaStream_t stream) {
    if (nrows == 0) return cudaSuccess;
    const int64_t cols = std::min<int64_t>((ne0 + 1023) / 1024, 65535);
    k_round_rows<<<dim3((unsigned)nrows, (unsigned)cols), 256, 0, stream>>>(bf16, src, (int)ne0, nb1, dst, stride);
    return cudaGetLastError();
}

}  // namespace gx

namespace {

static_assert(gx::kGroupedSmem == gx::kMaxSmem - 1024u, "the kernels' own shared memory");

// of allow_smem and resident_clusters
enum KernelSlot : int { kSlotGroup, kSlotLora, kSlotGmm, kSlotEnd = kSlotGmm + 6 };
static_assert(kSlotEnd <= kKernelSlots, "one slot per kernel");
int gmm_slot(int ctas, int mode) { return kSlotGmm + (ctas - 1) * 3 + mode; }

// The shared checks and the launch of the plain (up == NULL) and gated products.
int grouped_product(int type, const void * as, const void * up, int64_t ne00, int64_t ne01, int64_t nb01, int64_t nb02,
                    int64_t n_as, const void * b, int64_t ne11, int64_t nb11, const int32_t * offsets,
                    const int32_t * order, int64_t n_rows, int64_t gather, int scatter, int act, float alpha, float limit,
                    int type_dst, void * dst, int64_t nbd1, void * stream) {
    if (type != GX_TYPE_F16 && type != GX_TYPE_BF16) return GX_ERR_TYPE;
    const int out = out_kind(type_dst);
    if (out < 0) return GX_ERR_TYPE;
    if (act != GX_ACT_SWIGLU && act != GX_ACT_SWIGLU_OAI) return GX_ERR_INVALID;
    if (ne00 <= 0 || ne01 <= 0 || n_as <= 0 || ne11 < 0 || n_rows < 0 || gather < 0 || scatter < 0 || scatter > 1)
        return GX_ERR_INVALID;
    if (n_as > gx::kGroupMaxGroups || ne00 > kMaxSize || ne01 > kMaxSize || ne11 > kMaxSize || n_rows > kMaxSize ||
        gather > kMaxIndex)
        return GX_ERR_INVALID;
    if (n_rows == 0) return GX_OK;
    if (as == nullptr || b == nullptr || offsets == nullptr || dst == nullptr || ne11 == 0) return GX_ERR_INVALID;
    if (order == nullptr && (gather != 0 || scatter != 0)) return GX_ERR_INVALID;
    if (gather == 0 && ne11 < n_rows) return GX_ERR_INVALID;
    const int64_t esz = type_dst == GX_TYPE_F32 ? 4 : 2;
    if (nb01 < 0 || nb02 < 0 || nb11 < 0 || nbd1 < 0 || nb01 >= kMaxStride || nb02 >= kMaxStride ||
        nb11 >= kMaxStride)
        return GX_ERR_INVALID;
    if (n_as == 1) nb02 = nb01;                    // (never used to reach a second expert)
    if (nb01 % 16 || nb02 % 16 || nb11 % 16 || misaligned(as, 16) || misaligned(b, 16) || (up && misaligned(up, 16)))
        return GX_ERR_ALIGN;
    if (nbd1 % esz || misaligned(dst, esz) || misaligned(offsets, 4) || (order && misaligned(order, 4))) return GX_ERR_ALIGN;
    if (nb01 < 2 * ne00 || (n_as > 1 && !rows_fit(ne01, nb01, 2 * ne00, nb02)) || nb11 < 2 * ne00 || nbd1 < esz * ne01)
        return GX_ERR_INVALID;
    const bool glu = up != nullptr;

    gx::GmmParams p{};
    p.bf16 = type == GX_TYPE_BF16;
    p.offsets = offsets;
    p.order = order;
    p.G = (int32_t)n_as;
    p.n_rows = (int32_t)n_rows;
    p.x_rows = (int32_t)ne11;
    p.N = (int32_t)ne01;
    p.K = (int32_t)ne00;
    p.gather = (int32_t)gather;
    p.scatter = scatter;
    p.out = out;
    p.dst = static_cast<uint8_t *>(dst);
    p.nbd1 = nbd1;
    p.act = act;
    p.alpha = alpha;
    p.limit = limit;
    const int64_t touched = std::min(n_rows, n_as);
    const int64_t avg = (n_rows + touched - 1) / touched;
    // Pairs from 96 rows a group on average. Equal groups, gated, single CTAs and
    // pairs in us: K 2048, N 1024, 64 experts: 64 rows 96.5 and 95.9, 96 rows
    // 100.9 and 102.1, 192 rows 183 and 118; K 4096, N 1536: 96 rows 296 and 289,
    // 192 rows 595 and 321. (The average is all the host knows: groups of 2048
    // rows in 8 of 256 slots pass for 64 rows and take 235 us, as 8 experts 169.)
    const int ctas = avg >= 96 ? 2 : 1;
    const int64_t nk = (ne00 + gx::kGmmK - 1) / gx::kGmmK;
    // Where sums are long for the result's type, an accumulator takes 512
    // elements and the sums of the accumulators are rounded adds. A third of
    // TMEM holds them.
    p.seg = long_sum(out, ne00) ? 8 : 0;
    p.nt = 32;
    const int mode = !glu ? gx::GMM_PLAIN : ctas == 2 && p.seg == 0 ? gx::GMM_DUAL : gx::GMM_GLU;
    if (ctas == 2) p.nt = p.seg ? 160 : 256;
    else
        while (p.nt < 128 && p.nt < 2 * avg) p.nt *= 2;
    p.acc = p.seg ? p.nt : 256;
    const int sms = device_sms();
    if (sms == 0) return GX_ERR_CUDA;
    p.box = std::min(128, p.nt / ctas);
    const int out_rows = gx::gmm_out_rows(mode) * ctas;
    p.mt = (int32_t)((ne01 + out_rows - 1) / out_rows);
    const void * fn = mode == gx::GMM_DUAL ? (const void *)gx::k_gmm<2, gx::GMM_DUAL, gx::GMM_TILES>
                      : ctas == 2 ? (glu ? (const void *)gx::k_gmm<2, gx::GMM_GLU, gx::GMM_TILES>
                                         : (const void *)gx::k_gmm<2, gx::GMM_PLAIN, gx::GMM_TILES>)
                                  : (glu ? (const void *)gx::k_gmm<1, gx::GMM_GLU, gx::GMM_TILES>
                                         : (const void *)gx::k_gmm<1, gx::GMM_PLAIN, gx::GMM_TILES>);
    const int slot = gmm_slot(ctas, mode);
    cudaError_t e = allow_smem(fn, slot, gx::kGroupedSmem);
    if (e != cudaSuccess) return cuda_status(e);
    // The last round of tiles, when it leaves most SMs idle, is shared by the
    // CTAs of clusters that split K: pairs, or four or eight when not even one
    // round is full.
    p.split = 1;
    int64_t clusters = sms / ctas;
    if (ctas == 1 && p.nt == 32) {
        const int64_t tiles = (int64_t)p.mt * touched;
        for (int c = 8; c > 1; c /= 2) {
            const int64_t n = nk >= 4 * c ? resident_clusters(fn, c, gx::gmm_threads(mode), gx::kGroupedSmem, slot) : 0;
            if (n == 0 || (c > 2 && tiles > n)) continue;
            p.split = c;
            clusters = n;
            break;
        }
    }
    p.stages = gx::gmm_stages(ctas, p.nt, mode, p.G, p.split);
    if (p.stages < 2) return GX_ERR_INVALID;
    const uint32_t smem = gx::kGroupedAlign + (uint32_t)p.stages * gx::gmm_stage_bytes(ctas, p.nt, mode) +
                          gx::gmm_fixed_bytes(p.nt, mode, p.G, p.split);
    if (!encode_rows(&p.wmap, p.bf16, as, ne00, ne01, nb01, n_as, nb02, (uint32_t)gx::gmm_out_rows(mode)) ||
        (glu && !encode_rows(&p.umap, p.bf16, up, ne00, ne01, nb01, n_as, nb02, (uint32_t)gx::gmm_out_rows(mode))) ||
        !encode_rows(&p.xmap, p.bf16, b, ne00, ne11, nb11, 0, 0, gather ? 1u : (uint32_t)p.box))
        return GX_ERR_ALIGN;
    p.most = (int32_t)(n_rows / p.nt + touched);
    const int64_t most = (int64_t)p.mt * p.most;
    if (most > kMaxSize) return GX_ERR_INVALID;        // (a CTA's next tile is an index too)
    cudaLaunchConfig_t cfg{};
    const int cluster = ctas * p.split;
    cfg.gridDim = dim3((unsigned)(cluster * std::min<int64_t>(clusters, most)));
    cfg.blockDim = dim3((unsigned)gx::gmm_threads(mode));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    void * args[] = {&p};
    return cuda_status(cudaLaunchKernelExC(&cfg, fn, args));
}

}  // namespace

extern "C" {

int gx_group_rows(const int32_t * ids, int64_t ne20, int64_t ne21, int64_t nbi1, const int32_t * adapter, int64_t n_as,
                  int64_t n_adapters, int32_t * order, int32_t * offsets, void * stream) {
    if (ne20 <= 0 || ne21 < 0 || n_as <= 0 || n_adapters < 0) return GX_ERR_INVALID;
    if (offsets == nullptr) return GX_ERR_INVALID;
    if (ne21 > 0) {
        if (order == nullptr || (adapter == nullptr) != (n_adapters == 0)) return GX_ERR_INVALID;
        if (ids == nullptr && (adapter == nullptr || ne20 != 1 || n_as != 1)) return GX_ERR_INVALID;
    }
    if (ids != nullptr && (nbi1 < 4 * ne20 || nbi1 % 4)) return GX_ERR_INVALID;
    if (n_as > gx::kGroupMaxGroups || n_adapters > gx::kGroupMaxGroups) return GX_ERR_INVALID;
    const int64_t G = n_as * std::max<int64_t>(1, n_adapters);
    if (G > gx::kGroupMaxGroups || ne20 > kMaxIndex || ne21 > kMaxIndex || ne20 * ne21 > kMaxSize) return GX_ERR_INVALID;
    if (misaligned(order, 4) || misaligned(offsets, 4) || misaligned(ids, 4) || misaligned(adapter, 4)) return GX_ERR_ALIGN;
    gx::GroupParams p{};
    p.ids = ids;
    p.nbi1 = nbi1;
    p.adapter = adapter;
    p.k = (int32_t)ne20;
    p.n_as = (int32_t)n_as;
    p.n_adapters = (int32_t)n_adapters;
    p.G = (int32_t)G;
    p.P = (int32_t)(ne20 * ne21);
    // exact for dividends below 2^31: l = ceil(log2 k), m = floor(2^32 (2^l - k) / k) + 1
    while ((1ll << p.div_l) < ne20) ++p.div_l;
    p.div_m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << p.div_l) - (uint64_t)ne20)) / (uint64_t)ne20 + 1);
    p.order = order;
    p.offsets = offsets;
    const uint32_t bins = (uint32_t)(G + 1) * 4u;
    const int ncta = p.P <= 512 ? 1 : gx::kGroupCluster;      // (at 2048 pairs one CTA takes 6.3 us, eight 4.7)
    const int most = (int)std::min<uint32_t>(32u, (gx::kGroupSmem - 2u * bins) / bins);
    const int64_t steps = ((int64_t)p.P + 31) / 32;
    p.warps = (int)std::max<int64_t>(1, std::min<int64_t>(most, (steps + ncta - 1) / ncta));
    p.seg = (int)((steps + (int64_t)ncta * p.warps - 1) / ((int64_t)ncta * p.warps) * 32);
    const int threads = std::max(32 * p.warps, G > 1024 ? 1024 : 256);
    const uint32_t smem = (2u + (uint32_t)p.warps) * bins;
    cudaError_t e = allow_smem((const void *)gx::k_group_rows, kSlotGroup, gx::kGroupSmem);
    if (e != cudaSuccess) return cuda_status(e);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ncta);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)ncta;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, gx::k_group_rows, p));
}

int gx_mul_mat_grouped(int type, const void * as, int64_t ne00, int64_t ne01, int64_t nb01, int64_t nb02, int64_t n_as,
                       const void * b, int64_t ne11, int64_t nb11, const int32_t * offsets, const int32_t * order,
                       int64_t n_rows, int64_t gather, int scatter, int type_dst, void * dst, int64_t nbd1,
                       void * stream) {
    return grouped_product(type, as, nullptr, ne00, ne01, nb01, nb02, n_as, b, ne11, nb11, offsets, order, n_rows, gather,
                           scatter, GX_ACT_SWIGLU, 0.0f, 0.0f, type_dst, dst, nbd1, stream);
}

int gx_mul_mat_grouped_glu(int type, const void * gate, const void * up, int64_t ne00, int64_t ne01, int64_t nb01,
                           int64_t nb02, int64_t n_as, const void * b, int64_t ne11, int64_t nb11,
                           const int32_t * offsets, const int32_t * order, int64_t n_rows, int64_t gather, int scatter,
                           int act, float alpha, float limit, int type_dst, void * dst, int64_t nbd1, void * stream) {
    if (up == nullptr && n_rows > 0) return GX_ERR_INVALID;
    return grouped_product(type, gate, up, ne00, ne01, nb01, nb02, n_as, b, ne11, nb11, offsets, order, n_rows, gather,
                           scatter, act, alpha, limit, type_dst, dst, nbd1, stream);
}

int gx_lora_mul_mat(const gx_lora_desc * d, const void * x, int64_t ne11, int64_t nb11, const int32_t * offsets,
                    const int32_t * order, int64_t n_rows, int64_t gather, int type_dst, const void * base, int64_t nbb,
                    void * dst, int64_t nbd, void * stream) {
    if (d == nullptr) return GX_ERR_INVALID;
    if (d->type != GX_TYPE_F16 && d->type != GX_TYPE_BF16) return GX_ERR_TYPE;
    const int out = out_kind(type_dst);
    if (out < 0) return GX_ERR_TYPE;
    const int64_t K = d->ne00, N = d->ne01;
    int64_t nba2 = d->nba2, nbb2 = d->nbb2;
    if (K <= 0 || N <= 0 || d->rank <= 0 || d->rank > GX_LORA_MAX_RANK || d->n_as <= 0 || d->n_adapters <= 0 || ne11 < 0 ||
        n_rows < 0 || gather <= 0)
        return GX_ERR_INVALID;
    if (d->n_as > gx::kGroupMaxGroups || d->n_adapters > gx::kGroupMaxGroups || K > kMaxSize || N > kMaxSize ||
        ne11 > kMaxSize || n_rows > kMaxSize || gather > kMaxIndex)
        return GX_ERR_INVALID;
    const int64_t G = d->n_as * d->n_adapters;
    if (G > gx::kGroupMaxGroups) return GX_ERR_INVALID;
    if (n_rows == 0) return GX_OK;
    if (d->a == nullptr || d->b == nullptr || x == nullptr || offsets == nullptr || base == nullptr || dst == nullptr || ne11 == 0)
        return GX_ERR_INVALID;
    const int64_t esz = type_dst == GX_TYPE_F32 ? 4 : 2;
    if (d->nba1 < 0 || nba2 < 0 || d->nbb1 < 0 || nbb2 < 0 || nb11 < 0 || nbb < 0 || nbd < 0 || d->nba1 >= kMaxStride ||
        nba2 >= kMaxStride || d->nbb1 >= kMaxStride || nbb2 >= kMaxStride || nb11 >= kMaxStride)
        return GX_ERR_INVALID;
    if (G == 1) {                                      // (never used to reach a second adapter)
        nba2 = d->nba1;
        nbb2 = d->nbb1;
    }
    if (d->nba1 % 16 || nba2 % 16 || d->nbb1 % 16 || nbb2 % 16 || nb11 % 16 || misaligned(d->a, 16) || misaligned(d->b, 16) ||
        misaligned(x, 16))
        return GX_ERR_ALIGN;
    if (nbb % esz || nbd % esz || misaligned(base, esz) || misaligned(dst, esz) || misaligned(offsets, 4) ||
        misaligned(order, 4) || misaligned(d->ranks, 4) || misaligned(d->scale, 4))
        return GX_ERR_ALIGN;
    if (d->nba1 < 2 * K || d->nbb1 < 2 * d->rank || nb11 < 2 * K || nbb < esz * N || nbd < esz * N) return GX_ERR_INVALID;
    if (G > 1 && (!rows_fit(d->rank, d->nba1, 2 * K, nba2) || !rows_fit(N, d->nbb1, 2 * d->rank, nbb2))) return GX_ERR_INVALID;

    gx::LoraParams p{};
    p.offsets = offsets;
    p.order = order;
    p.ranks = d->ranks;
    p.scale = d->scale;
    p.base = static_cast<const uint8_t *>(base);
    p.dst = static_cast<uint8_t *>(dst);
    p.nbb = nbb;
    p.nbd = nbd;
    p.G = (int32_t)G;
    p.n_as = (int32_t)d->n_as;
    p.n_rows = (int32_t)n_rows;
    p.x_rows = (int32_t)ne11;
    p.gather = (int32_t)gather;
    p.N = (int32_t)N;
    p.K = (int32_t)K;
    p.rank = (int32_t)d->rank;
    p.ra = 16;
    while (p.ra < p.rank) p.ra *= 2;
    p.bf16 = d->type == GX_TYPE_BF16;
    p.out = out;
    p.copy = base != dst;
    p.seg = long_sum(out, K) ? gx::kLoraSeg : 0;
    if (p.copy == 0 && nbb != nbd) return GX_ERR_INVALID;
    if (!encode_rows(&p.amap, p.bf16, d->a, K, d->rank, d->nba1, G, nba2, (uint32_t)p.ra) ||
        !encode_rows(&p.bmap, p.bf16, d->b, d->rank, N, d->nbb1, G, nbb2, 128u, (uint32_t)std::min(p.ra, 64)) ||
        !encode_rows(&p.xmap, p.bf16, x, K, ne11, nb11, 0, 0, 1u) ||
        !encode_rows(&p.rmap, p.bf16, x, K, ne11, nb11, 0, 0, (uint32_t)gx::kLoraRows))
        return GX_ERR_ALIGN;
    const int sms = device_sms();
    if (sms == 0) return GX_ERR_CUDA;
    const int per_sm = gx::lora_ctas_per_sm(p.ra, p.G);
    p.stages = gx::lora_stages(p.ra, p.G);
    if (p.stages < 2) return GX_ERR_INVALID;
    const uint32_t smem = gx::kGroupedAlign + (uint32_t)p.stages * gx::lora_stage_bytes(p.ra) + gx::lora_fixed_bytes(p.ra, p.G);
    const int64_t most = n_rows / gx::kLoraRows + std::min(n_rows, G);
    p.most = (int32_t)(n_rows / gx::kLoraRows + std::min(n_rows, G + 1));
    cudaError_t e = allow_smem((const void *)gx::k_lora, kSlotLora, gx::kGroupedSmem);
    if (e != cudaSuccess) return cuda_status(e);
    // A cluster per tile of rows, of the size whose rounds of tiles cost least:
    // a tile's work is shared by its CTAs, but for about a sixteenth that each
    // repeats. (Whether or not base is dst: the split of K sets the result's
    // bits.) In us with 1, 2, 4 and 8 CTAs, BF16, f32 results, the choice marked:
    // 1 row, rank 16, K = N = 2048: 25.5, 16.9, 12.7, 11.4*; 64 rows of 48
    // adapters, rank 64, K = N = 4096: 49.5, 29.5, 21.1*, 31.2; 4096 rows of 128,
    // rank 16, K 2048, N 768: 24.1*, 27.2, 35.0, 67.9.
    int ctas = 1;
    int64_t clusters = (int64_t)sms * per_sm, best = 0;
    for (int c = 1; c <= 8 && (c == 1 || c <= std::max((K + 127) / 128, (N + 127) / 128)); c *= 2) {
        const int64_t n = c == 1 ? clusters
                                 : resident_clusters((const void *)gx::k_lora, c, gx::kLoraThreads, gx::kGroupedSmem, kSlotLora) * per_sm;
        if (n == 0) break;
        const int64_t cost = (most + n - 1) / n * (16 / c + 1);
        if (c == 1 || cost < best) {
            best = cost;
            ctas = c;
            clusters = n;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(ctas * std::min<int64_t>(clusters, most + (p.copy ? n_rows / gx::kLoraRows + 1 : 0))));
    cfg.blockDim = dim3(gx::kLoraThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)ctas;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, gx::k_lora, p));
}

}  // extern "C"
