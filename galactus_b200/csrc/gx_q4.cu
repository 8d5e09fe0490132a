// Entry points of the products with 4-bit weights and of the norms around a
// block. No C++ exception crosses this boundary; every entry point returns GX_*.
#include <algorithm>

#include "gx_block.cuh"
#include "gx_kernels.h"
#include "gx_launch.h"
#include "gx_q4.cuh"

namespace gx {

cudaError_t read_and_clear_q4_error(int * code) {
    int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(code, g_dev_error, sizeof(int));
    if (e != cudaSuccess) return e;
    return cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(int));
}

}  // namespace gx

namespace {

enum KernelSlot : int { kSlotQ4 = 0, kSlotRows = 8, kSlotTiles = kSlotRows + 6, kSlotEnd = kSlotTiles + 8 };
static_assert(kSlotEnd <= kKernelSlots, "one slot per kernel");
static_assert(gx::kQ4MaxIds == GX_Q4_MAX_IDS && gx::kBlockMaxWidth == GX_BLOCK_MAX_WIDTH, "limits of the header");

// Rows of a group above which matrix tiles are made for the tensor cores. In us
// with 16, 24, 32 and 48 rows: 64 tokens x 8 of 128 experts, 1536 x 4096, 117, 121,
// 125, 124; 1031 tokens x 8 of 64, 1024 x 2048, 172, 172, 176, 180; gated, 2048 tokens
// x 8 of 128, 4096 x 1536, 1001, 1010, 1013, 1032; one matrix of 4096 x 14336 with 32
// rows 44, 45, 56, 55. (16 and 24 differ by as much as a case does from run to run;
// below the border no sum is of a weight's parts.)
constexpr int64_t kTileRows = 24;

// A launch that may begin while the kernel before it on the stream ends: the
// kernels wait (griddepcontrol.wait) before they read or write anything.
template <typename P>
cudaError_t launch_next(const void * fn, dim3 grid, int threads, uint32_t smem, int cluster, void * stream, P & p) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    void * args[] = {&p};
    return cudaLaunchKernelExC(&cfg, fn, args);
}

template <bool BF16, bool Q41>
const void * q4_kernel(bool glu) {
    return glu ? (const void *)gx::k_q4<BF16, Q41, true> : (const void *)gx::k_q4<BF16, Q41, false>;
}
const void * q4_kernel(bool bf16, bool q41, bool glu) {
    return bf16 ? (q41 ? q4_kernel<true, true>(glu) : q4_kernel<true, false>(glu))
                : (q41 ? q4_kernel<false, true>(glu) : q4_kernel<false, false>(glu));
}

template <int MODE>
const void * q4_tiles_kernel(bool bf16, bool q41) {
    if (q41) return bf16 ? (const void *)gx::k_gmm<2, MODE, gx::GMM_Q4_1_BF16> : (const void *)gx::k_gmm<2, MODE, gx::GMM_Q4_1_F16>;
    return bf16 ? (const void *)gx::k_gmm<2, MODE, gx::GMM_Q4_0_BF16> : (const void *)gx::k_gmm<2, MODE, gx::GMM_Q4_0_F16>;
}

// rows of blocks as 32-bit words, boxes of `words` by `rows`
bool encode_blocks(CUtensorMap * map, const void * base, bool q41, int64_t K, int64_t N, int64_t nb1, int64_t mats, int64_t nb2, uint32_t words,
                   uint32_t rows) {
    const auto enc = map_encoder();
    if (enc == nullptr) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)(K / 64 * (q41 ? 10 : 9)), (cuuint64_t)N, (cuuint64_t)mats};
    const cuuint64_t strides[2] = {(cuuint64_t)nb1, (cuuint64_t)nb2};
    const cuuint32_t boxes[3] = {words, rows, 1u};
    const cuuint32_t elem[3] = {1u, 1u, 1u};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void *>(base), dims, strides, boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Many rows per matrix: the grouped products' kernel on CTA pairs, its matrix
// tiles made from the blocks.
int q4_tiles(gx::GmmParams & p, bool q41, bool glu, const void * b, int64_t nb11, int64_t touched, void * stream) {
    const int mode = glu ? gx::GMM_GLU : gx::GMM_PLAIN;
    // Parts of 16 bits that a weight is made of: d (q - 8) whole, d q + m to 22 bits
    // (F16) or to 16, and for f32 results 24 (BF16). One part, a weight rounded to the
    // rows' type, would leave results of 16 bits 1.7 times as far from 64 bits.
    p.parts = p.out == gx::GMM_F32 && q41 && p.bf16 ? 3 : 2;
    // (two MMAs a chunk: sums of 256 elements where grouped products take 512)
    p.seg = long_sum(p.out, 2 * (int64_t)p.K) ? 4 : 0;
    p.nt = p.seg ? 160 : 256;
    while (gx::gmm_q4_stages(q41, p.nt, mode, p.G, p.parts) < 2) p.nt -= 32;       // (thousands of matrices, f32 results)
    p.acc = p.seg ? p.nt : 256;
    p.box = p.nt / 2;
    if (!encode_rows(&p.xmap, p.bf16 != 0, b, p.K, p.x_rows, nb11, 0, 0, p.gather ? 1u : (uint32_t)p.box)) return GX_ERR_ALIGN;
    // rows on 16 bytes come as boxes of 32 rows by a stage's words
    p.boxes = p.nb01 % 16 == 0 && p.nb02 % 16 == 0 && encode_blocks(&p.wmap, p.w0, q41, p.K, p.N, p.nb01, p.G, p.nb02, gx::gmm_q4_pitch(q41) / 4u, 32u) &&
              (!glu || encode_blocks(&p.umap, p.w1, q41, p.K, p.N, p.nb01, p.G, p.nb02, gx::gmm_q4_pitch(q41) / 4u, 32u));
    p.split = 1;
    const int out_rows = gx::gmm_out_rows(mode) * 2;
    p.mt = (int32_t)((p.N + out_rows - 1) / out_rows);
    p.most = (int32_t)(p.n_rows / p.nt + touched);
    const int64_t most = (int64_t)p.mt * p.most;
    if (most > kMaxSize) return GX_ERR_INVALID;
    const int sms = device_sms();
    if (sms == 0) return GX_ERR_CUDA;
    const void * fn = glu ? q4_tiles_kernel<gx::GMM_GLU>(p.bf16 != 0, q41) : q4_tiles_kernel<gx::GMM_PLAIN>(p.bf16 != 0, q41);
    cudaError_t e = allow_smem(fn, kSlotTiles + (glu ? 4 : 0) + (q41 ? 2 : 0) + (p.bf16 ? 1 : 0), gx::kGroupedSmem);
    if (e != cudaSuccess) return cuda_status(e);
    p.stages = gx::gmm_q4_stages(q41, p.nt, mode, p.G, p.parts);
    const uint32_t smem = gx::kGroupedAlign + (uint32_t)p.stages * gx::gmm_q4_stage_bytes(p.nt, p.parts) + gx::gmm_q4_fixed_bytes(q41, p.nt, mode, p.G);
    return cuda_status(launch_next(fn, dim3((unsigned)(2 * std::min<int64_t>(sms / 2, most))), gx::gmm_q4_threads(mode), smem,
                                   2, stream, p));
}

// The shared checks and the launch of the plain (up == NULL) and gated products.
int q4_product(int type, const void * as, const void * up, int64_t ne00, int64_t ne01, int64_t nb01, int64_t nb02, int64_t n_as,
               int type_b, const void * b, int64_t ne11, int64_t nb11, const int32_t * ids, const int32_t * offsets,
               const int32_t * order, int64_t n_rows, int64_t gather, int scatter, int act, float alpha, float limit, int type_dst,
               void * dst, int64_t nbd1, void * stream) {
    if (type != GX_TYPE_Q4_0 && type != GX_TYPE_Q4_1) return GX_ERR_TYPE;
    if (type_b != GX_TYPE_F16 && type_b != GX_TYPE_BF16) return GX_ERR_TYPE;
    const int out = out_kind(type_dst);
    if (out < 0) return GX_ERR_TYPE;
    if (act != GX_ACT_SWIGLU && act != GX_ACT_SWIGLU_OAI) return GX_ERR_INVALID;
    if (ne00 <= 0 || ne01 <= 0 || n_as <= 0 || ne11 < 0 || n_rows < 0 || gather < 0 || scatter < 0 || scatter > 1)
        return GX_ERR_INVALID;
    if (n_as > gx::kGroupMaxGroups || ne00 > GX_Q4_MAX_K || ne01 > kMaxSize || ne11 > kMaxSize || n_rows > kMaxSize ||
        gather > kMaxIndex)
        return GX_ERR_INVALID;
    if (ids != nullptr && (offsets != nullptr || order != nullptr || n_rows > GX_Q4_MAX_IDS)) return GX_ERR_INVALID;
    if (n_rows == 0) return GX_OK;
    if (as == nullptr || b == nullptr || dst == nullptr || ne11 == 0) return GX_ERR_INVALID;
    if (ids == nullptr && offsets == nullptr && n_as != 1) return GX_ERR_INVALID;
    if (ids != nullptr) {
        scatter = 1;
        gather = std::max<int64_t>(1, gather);
    } else if (order == nullptr && (gather != 0 || scatter != 0)) {
        return GX_ERR_INVALID;
    }
    if ((gather == 0 || (ids != nullptr && gather == 1)) && ne11 < n_rows) return GX_ERR_INVALID;
    const int64_t esz = type_dst == GX_TYPE_F32 ? 4 : 2;
    if (nb01 < 0 || nb02 < 0 || nb11 < 0 || nbd1 < 0 || nb01 >= kMaxStride || nb02 >= kMaxStride || nb11 >= kMaxStride)
        return GX_ERR_INVALID;
    if (n_as == 1) nb02 = nb01;                    // (never used to reach a second expert)
    if (ne00 % 64 || nb01 % 4 || nb02 % 4 || nb11 % 16 || misaligned(as, 16) || misaligned(b, 16) || (up && misaligned(up, 16)))
        return GX_ERR_ALIGN;
    if (nbd1 % esz || misaligned(dst, esz) || misaligned(ids, 4) || misaligned(offsets, 4) || misaligned(order, 4))
        return GX_ERR_ALIGN;
    const int64_t row = gx::row_bytes(type, ne00);
    if (nb01 < row || (n_as > 1 && !rows_fit(ne01, nb01, row, nb02)) || nb11 < 2 * ne00 || nbd1 < esz * ne01) return GX_ERR_INVALID;
    const bool glu = up != nullptr, q41 = type == GX_TYPE_Q4_1, bf16 = type_b == GX_TYPE_BF16;

    gx::Q4Params p{};
    p.w0 = static_cast<const uint8_t *>(as);
    p.w1 = static_cast<const uint8_t *>(glu ? up : as);
    p.nb01 = nb01;
    p.nb02 = nb02;
    p.x = static_cast<const uint8_t *>(b);
    p.nb11 = nb11;
    p.ids = ids;
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
    // Groups of more than kTileRows rows go to the tensor cores' tiles, shorter ones
    // (which only the device tells apart) stream their matrices past a few rows.
    if (ids == nullptr && n_rows > kTileRows) {
        gx::GmmParams t{};
        t.bf16 = bf16;
        t.offsets = offsets;
        t.order = order;
        t.G = p.G;
        t.n_rows = p.n_rows;
        t.x_rows = p.x_rows;
        t.N = p.N;
        t.K = p.K;
        t.gather = p.gather;
        t.scatter = p.scatter;
        t.out = out;
        t.dst = p.dst;
        t.nbd1 = nbd1;
        t.act = act;
        t.alpha = alpha;
        t.limit = limit;
        t.w0 = p.w0;
        t.w1 = p.w1;
        t.nb01 = nb01;
        t.nb02 = nb02;
        t.lo = offsets != nullptr ? (int32_t)kTileRows + 1 : 1;
        const int rc = q4_tiles(t, q41, glu, b, nb11, touched, stream);
        if (rc != GX_OK || offsets == nullptr) return rc;
    }
    const gx::Q4Shape shape = gx::q4_shape(q41, ne00, n_rows);
    p.warps = shape.warps;
    p.cap = shape.cap;
    p.buffers = shape.buffers;
    p.lo = 1;
    p.hi = ids == nullptr ? (int32_t)kTileRows : (int32_t)kMaxIndex;
    const int rows = (glu ? 8 : 16) * gx::kQ4Mt;
    p.rt = (int32_t)((ne01 + rows - 1) / rows);
    const int64_t tiles = n_rows / p.cap + touched, most = p.rt * tiles;
    if (tiles > kMaxSize || most > kMaxSize) return GX_ERR_INVALID;
    p.most = (int32_t)tiles;
    const int sms = device_sms();
    if (sms == 0) return GX_ERR_CUDA;
    // Warps that share K: as many as leave four fifths of the jobs a team each. In
    // us with 2, 4, 8 and 16 of 16 warps, one row, the choice marked: 512 jobs of 12
    // pairs of blocks 10.9, 9.4*, 11.0, 12.7; 720 of 45: 30, 23*, 24, 26; 448 of 64:
    // 19.1, 17.8*, 18.5, 20.3; 128 of 64: 16.9, 11.2, 8.5, 8.3*.
    const int64_t jobs = p.rt * (touched + (n_rows - touched) / p.cap);
    p.share = 2;
    for (int c = 4; c <= p.warps; c += 2)
        if (p.warps % c == 0 && (int64_t)sms * (p.warps / c) * 5 >= jobs * 4) p.share = c;
    const uint32_t words = (uint32_t)gx::q4_pitch(q41) / 4u, box = glu ? 16u : 32u;
    p.boxes = nb01 % 16 == 0 && nb02 % 16 == 0 && encode_blocks(&p.wmap, p.w0, q41, ne00, ne01, nb01, n_as, nb02, words, box) &&
              (!glu || encode_blocks(&p.umap, p.w1, q41, ne00, ne01, nb01, n_as, nb02, words, box));
    const void * fn = q4_kernel(bf16, q41, glu);
    const int slot = kSlotQ4 + (bf16 ? 4 : 0) + (q41 ? 2 : 0) + (glu ? 1 : 0);
    cudaError_t e = allow_smem(fn, slot, gx::kQ4Smem);
    if (e != cudaSuccess) return cuda_status(e);
    const int64_t grid = std::min<int64_t>(sms, (most * p.share + p.warps - 1) / p.warps);
    return cuda_status(launch_next(fn, dim3((unsigned)grid), 32 * p.warps, gx::q4_smem(q41, ne00, p.warps, p.cap, p.buffers), 1, stream,
                                   p));
}

// rows of ne0 elements of a result type: as the kernel takes them; false: a bad type, stride or alignment (in rc)
bool block_rows(int type, const void * p, int64_t ne0, int64_t nb, int64_t ne1, gx::BlockRows & out, bool & vec, int & rc) {
    out = gx::BlockRows{nullptr, 0, 0};
    if (p == nullptr) return true;
    const int kind = out_kind(type);
    if (kind < 0) {
        rc = GX_ERR_TYPE;
        return false;
    }
    const int64_t esz = kind == gx::GMM_F32 ? 4 : 2;
    if (nb < 0 || nb >= kMaxStride || (ne1 > 1 && nb < esz * ne0)) {
        rc = GX_ERR_INVALID;
        return false;
    }
    if (nb % esz || misaligned(p, esz)) {
        rc = GX_ERR_ALIGN;
        return false;
    }
    vec = vec && !misaligned(p, 16) && (ne1 <= 1 || nb % 16 == 0);
    out = gx::BlockRows{static_cast<uint8_t *>(const_cast<void *>(p)), nb, kind};
    return true;
}

constexpr uint32_t kStreamSmem = 220u * 1024u;
// Rows of fewer elements, or fewer elements in all, go a CTA each (k_block) rather
// than through rings (k_block_rows). In us a CTA each / rings, sum of k rows of
// BF16, residual, next norm: 8192 rows of 1024, k = 1, 27 / 34; of 2880, 109 / 52;
// of 512, k = 8, 42 / 77; of 2048, k = 8, 192 / 88. 296 and 592 rows of 4096, k = 1, 4.7 /
// 4.9 and 8.9 / 8.5; of 2048, k = 8, 5.6 / 6.3 and 14.2 / 11.0; 148 of 7168, k = 8, 13.0 / 6.6.
constexpr int kStreamWidth = 2048;
constexpr int64_t kStreamElements = 1 << 20;
// Steps of a lane up to which a row has a warp, with any number of rows and with
// many. In us a CTA each / a warp each, as above: 74 rows of 256, k = 1, 2.4 / 2.2;
// 8192, 13.0 / 6.3; 74 of 128, k = 8, 4.4 / 3.1; 592, 2368 and 8192 of 512, k = 1, 3.3 /
// 3.6, 5.6 / 5.1 and 17.1 / 13.7; 8192 of 1024, 27 / 29.
constexpr int kWarpSteps = 1, kWarpStepsMany = 2, kWarpMany = 2048;

template <int YT>
const void * block_kernel(bool vec, bool cluster) {
    constexpr int n = gx::kBlockUnits;
    return vec ? (cluster ? (const void *)gx::k_block<YT, true, gx::ROW_CLUSTER, n> : (const void *)gx::k_block<YT, true, gx::ROW_CTA, n>)
               : (cluster ? (const void *)gx::k_block<YT, false, gx::ROW_CLUSTER, n> : (const void *)gx::k_block<YT, false, gx::ROW_CTA, n>);
}
template <int YT>
const void * block_warp_kernel(int steps) {
    return steps == 1 ? (const void *)gx::k_block<YT, true, gx::ROW_WARP, 1> : (const void *)gx::k_block<YT, true, gx::ROW_WARP, kWarpStepsMany>;
}

template <int YT>
int launch_block_rows(gx::BlockParams & p, int grid, int warps, int slots, int slot_bytes, void * stream) {
    const void * fn = warps <= 8 ? (const void *)gx::k_block_rows<YT, 8> : (const void *)gx::k_block_rows<YT, gx::kRowsMaxWarps>;
    const uint32_t smem = (uint32_t)(slots * slot_bytes);
    cudaError_t e = allow_smem(fn, kSlotRows + YT + (warps <= 8 ? 0 : 3), kStreamSmem);
    if (e != cudaSuccess) return cuda_status(e);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)(32 * (warps + 1)));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    void * args[] = {&p, &slots, &slot_bytes};
    return cuda_status(cudaLaunchKernelExC(&cfg, fn, args));
}
int launch_block_rows(gx::BlockParams & p, int sms, void * stream) {
    const auto size = [](const gx::BlockRows & r) { return r.p == nullptr ? 0 : r.type == gx::GMM_F32 ? 4 : 2; };
    const int slot_bytes = (p.H * std::max(size(p.y), std::max(size(p.shared), size(p.res))) + 127) / 128 * 128;
    const int warps = (p.H + 32 * gx::kBlockUnit * gx::kBlockUnits - 1) / (32 * gx::kBlockUnit * gx::kBlockUnits);
    const int ctas = gx::rows_ctas(warps <= 8 ? 8 : gx::kRowsMaxWarps);
    const int slots = std::min<int>(gx::kRowsMaxSlots, (int)(kStreamSmem / ctas) / slot_bytes);
    const int grid = std::min<int64_t>((int64_t)sms * ctas, p.T);
    switch (p.y.type) {
        case gx::GMM_F32: return launch_block_rows<gx::GMM_F32>(p, grid, warps, slots, slot_bytes, stream);
        case gx::GMM_F16: return launch_block_rows<gx::GMM_F16>(p, grid, warps, slots, slot_bytes, stream);
        default: return launch_block_rows<gx::GMM_BF16>(p, grid, warps, slots, slot_bytes, stream);
    }
}

int launch_block(gx::BlockParams & p, bool vec, void * stream) {
    p.one = 1.0f;
    p.per = 1.0f / (float)p.H;
    const int sms = device_sms();
    if (sms == 0) return GX_ERR_CUDA;
    vec = vec && p.H % 8 == 0 && !misaligned(p.norm, 16) && !misaligned(p.next_norm, 16) &&
          (p.gate_step == 0 || (!misaligned(p.gate, 16) && p.gate_nb % 16 == 0));
    const int units = (p.H + gx::kBlockUnit - 1) / gx::kBlockUnit;
    if (vec && p.k <= 32 && p.H <= gx::kRowsMaxWidth && p.H >= kStreamWidth && (int64_t)p.T * p.H >= kStreamElements)
        return launch_block_rows(p, sms, stream);
    const int steps = (units + 31) / 32;
    if (vec && steps <= (p.T >= kWarpMany ? kWarpStepsMany : kWarpSteps)) {
        const void * fn = p.y.type == gx::GMM_F32   ? block_warp_kernel<gx::GMM_F32>(steps)
                          : p.y.type == gx::GMM_F16 ? block_warp_kernel<gx::GMM_F16>(steps)
                                                    : block_warp_kernel<gx::GMM_BF16>(steps);
        const int ctas = (p.T - 1) / gx::kBlockWarps + 1;
        return cuda_status(launch_next(fn, dim3((unsigned)ctas), 32 * gx::kBlockWarps, 0, 1, stream, p));
    }
    // A cluster per row: where a CTA's registers do not hold the row, or where few rows
    // leave SMs idle and a CTA's threads would take two steps. One row, us without and
    // with: 2880 elements 2.7, 2.9; 4096 3.0, 2.9; 5120 3.5, 3.0; 7168, k = 8, 7.5, 4.7.
    int cluster = 1;
    while (cluster < gx::kBlockMaxCluster &&
           (units > cluster * gx::kBlockUnits * gx::kBlockMaxThreads ||
            ((int64_t)p.T * cluster * 2 <= sms && units > gx::kBlockMaxThreads && units > cluster * 64)))
        cluster *= 2;
    const int per = (units + cluster - 1) / cluster;
    // Steps of a thread: one, or two where CTAs wait for SMs and there is one row to
    // load (290 rows of 2880, k = 1: 5.0 us with one, 3.7 with two; of 2048, k = 8: 4.9, 8.1)
    int threads = 64;
    while (threads < gx::kBlockMaxThreads && threads * (p.k == 1 && p.T * cluster > sms ? gx::kBlockUnits : 1) < per) threads *= 2;
    const int kind = p.y.type;
    const void * fn = kind == gx::GMM_F32   ? block_kernel<gx::GMM_F32>(vec, cluster > 1)
                      : kind == gx::GMM_F16 ? block_kernel<gx::GMM_F16>(vec, cluster > 1)
                                            : block_kernel<gx::GMM_BF16>(vec, cluster > 1);
    return cuda_status(launch_next(fn, dim3((unsigned)(p.T * cluster)), threads, 0, cluster, stream, p));
}

}  // namespace

extern "C" {

int gx_mul_mat_q4(int type, const void * as, int64_t ne00, int64_t ne01, int64_t nb01, int64_t nb02, int64_t n_as, int type_b,
                  const void * b, int64_t ne11, int64_t nb11, const int32_t * ids, const int32_t * offsets, const int32_t * order,
                  int64_t n_rows, int64_t gather, int scatter, int type_dst, void * dst, int64_t nbd1, void * stream) {
    return q4_product(type, as, nullptr, ne00, ne01, nb01, nb02, n_as, type_b, b, ne11, nb11, ids, offsets, order, n_rows, gather,
                      scatter, GX_ACT_SWIGLU, 0.0f, 0.0f, type_dst, dst, nbd1, stream);
}

int gx_mul_mat_q4_glu(int type, const void * gate, const void * up, int64_t ne00, int64_t ne01, int64_t nb01, int64_t nb02,
                      int64_t n_as, int type_b, const void * b, int64_t ne11, int64_t nb11, const int32_t * ids,
                      const int32_t * offsets, const int32_t * order, int64_t n_rows, int64_t gather, int scatter, int act,
                      float alpha, float limit, int type_dst, void * dst, int64_t nbd1, void * stream) {
    if (up == nullptr && n_rows > 0) return GX_ERR_INVALID;
    return q4_product(type, gate, up, ne00, ne01, nb01, nb02, n_as, type_b, b, ne11, nb11, ids, offsets, order, n_rows, gather,
                      scatter, act, alpha, limit, type_dst, dst, nbd1, stream);
}

int gx_rms_norm(int type_src, const void * src, int64_t ne0, int64_t ne1, int64_t nb1, const float * weight, float eps, int type_dst,
                void * dst, int64_t nbd1, void * stream) {
    if (ne0 <= 0 || ne0 > GX_BLOCK_MAX_WIDTH || ne1 < 0 || ne1 > kMaxSize / gx::kBlockMaxCluster || !(eps >= 0.0f)) return GX_ERR_INVALID;
    if (out_kind(type_src) < 0 || out_kind(type_dst) < 0) return GX_ERR_TYPE;
    if (ne1 == 0) return GX_OK;
    if (src == nullptr || dst == nullptr) return GX_ERR_INVALID;
    gx::BlockParams p{};
    bool vec = true;
    int rc = GX_OK;
    if (!block_rows(type_src, src, ne0, nb1, ne1, p.y, vec, rc) || !block_rows(type_dst, dst, ne0, nbd1, ne1, p.next, vec, rc)) return rc;
    if (misaligned(weight, 4)) return GX_ERR_ALIGN;
    p.H = (int32_t)ne0;
    p.T = (int32_t)ne1;
    p.k = 1;
    p.y_nb2 = nb1;
    p.scale = 1.0f;
    p.has_next = 1;
    p.next_eps = eps;
    p.next_norm = weight;
    return launch_block(p, vec, stream);
}

int gx_block_out(const gx_block_desc * d, void * stream) {
    if (d == nullptr) return GX_ERR_INVALID;
    if (d->ne0 <= 0 || d->ne0 > GX_BLOCK_MAX_WIDTH || d->ne1 < 0 || d->ne1 > kMaxSize / gx::kBlockMaxCluster || d->k <= 0 ||
        d->ne1 * (int64_t)d->k > kMaxSize)
        return GX_ERR_INVALID;
    if ((d->norm != nullptr && !(d->eps >= 0.0f)) || (d->next != nullptr && !(d->next_eps >= 0.0f))) return GX_ERR_INVALID;
    if (d->ne1 == 0) return GX_OK;
    if (d->y == nullptr || (d->dst == nullptr && d->next == nullptr)) return GX_ERR_INVALID;
    if (d->shared_gate != nullptr && d->shared == nullptr) return GX_ERR_INVALID;
    gx::BlockParams p{};
    bool vec = true;
    int rc = GX_OK;
    if (!block_rows(d->type_y, d->y, d->ne0, d->nby1, d->k, p.y, vec, rc)) return rc;
    gx::BlockRows tokens;
    if (!block_rows(d->type_y, d->y, d->ne0, d->nby2, d->ne1, tokens, vec, rc) ||
        !block_rows(d->type_shared, d->shared, d->ne0, d->nbs, d->ne1, p.shared, vec, rc) ||
        !block_rows(d->type_residual, d->residual, d->ne0, d->nbr, d->ne1, p.res, vec, rc) ||
        !block_rows(d->type_dst, d->dst, d->ne0, d->nbd, d->ne1, p.dst, vec, rc) ||
        !block_rows(d->type_next, d->next, d->ne0, d->nbn, d->ne1, p.next, vec, rc))
        return rc;
    if (misaligned(d->weights, 4) || misaligned(d->ids, 4) || misaligned(d->shared_gate, 4) || misaligned(d->norm, 4) ||
        misaligned(d->next_norm, 4) || misaligned(d->gate, 4))
        return GX_ERR_ALIGN;
    if (d->gate != nullptr) {
        if ((d->gne0 != 1 && d->gne0 != d->ne0) || d->nbg < 0 || d->nbg >= kMaxStride || (d->nbg != 0 && d->nbg < 4 * d->gne0))
            return GX_ERR_INVALID;
        if (d->gate_act != GX_GATE_NONE && d->gate_act != GX_GATE_SIGMOID) return GX_ERR_INVALID;
        if (d->nbg % 4) return GX_ERR_ALIGN;
        p.gate = d->gate;
        p.gate_nb = d->nbg;
        p.gate_step = d->gne0 == d->ne0 && d->ne0 > 1 ? 1 : 0;
        p.gate_sigmoid = d->gate_act == GX_GATE_SIGMOID;
    }
    p.H = (int32_t)d->ne0;
    p.T = (int32_t)d->ne1;
    p.k = d->k;
    p.y_nb2 = d->nby2;
    p.w = d->weights;
    p.ids = d->ids;
    p.shared_gate = d->shared_gate;
    p.norm = d->norm;
    p.has_norm = d->norm != nullptr;
    p.has_next = d->next != nullptr;
    p.eps = d->eps;
    p.next_eps = d->next_eps;
    p.scale = d->scale;
    p.next_norm = d->next_norm;
    return launch_block(p, vec, stream);
}

}  // extern "C"
