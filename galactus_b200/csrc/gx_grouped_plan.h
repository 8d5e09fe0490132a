// Tiles and shared memory of the kernels on grouped rows (plain C++, used by
// the kernels, by the entry points and by the host-side tests).
#pragma once

#include "gx_formats.h"

namespace gx {

// Dynamic shared memory that a launch may ask for: 227 KB less 1 KB for the
// barriers and lists that the kernels declare themselves. 1 KB of it goes into
// aligning the ring.
constexpr uint32_t kGroupedSmem = 226u * 1024u;
constexpr uint32_t kGroupedAlign = 1024u;

// ------------------------------------------------------------- products

constexpr int kGmmRows = 128;                  // matrix rows of an MMA per CTA: TMEM lanes
constexpr int kGmmK = 64;                      // elements of K per stage: one 128-byte swizzled row
constexpr uint32_t kGmmATile = kGmmRows * 128u;
constexpr int kGmmMaxStages = 12;
constexpr int kGmmGatherWarps = 4;             // 32 rows each
// what a kernel makes of its tiles
enum : int {
    GMM_PLAIN = 0,   // y = W x: 128 rows of W
    GMM_GLU = 1,     // gated: 64 gate and 64 up rows, two accumulators in turn
    GMM_DUAL = 2,    // gated, CTA pairs, 16-bit results: 128 gate and 128 up rows, one accumulator each
};
GX_HD constexpr int gmm_epi_warps(int mode) { return mode == GMM_DUAL ? 8 : 4; }
GX_HD constexpr int gmm_threads(int mode) { return 32 * (2 + kGmmGatherWarps + gmm_epi_warps(mode)); }
GX_HD constexpr int gmm_out_rows(int mode) { return mode == GMM_GLU ? 64 : 128; }
GX_HD constexpr uint32_t gmm_a_bytes(int mode) { return mode == GMM_DUAL ? 2u * kGmmATile : kGmmATile; }
constexpr uint32_t kGmmStaging = 4u * 32u * 32u * 4u;            // results of 32 (dual: 16) columns per epilogue warp
constexpr uint32_t kGmmXchg = 2u * 2u * 2u * 16u * 32u * 4u;   // gated: [buffer][warp pair][direction][column][lane] f32

// bytes of a ring stage: the matrix tile and the CTA's rows
GX_HD constexpr uint32_t gmm_stage_bytes(int ctas, int nt, int mode) {
    return gmm_a_bytes(mode) + (uint32_t)(nt / ctas) * 128u;
}
// and of everything behind the ring
GX_HD constexpr uint32_t gmm_fixed_bytes(int nt, int mode, int groups, int split) {
    return (uint32_t)(groups + 1) * 4u + kGmmStaging + (mode == GMM_GLU ? kGmmXchg : 0u) +
           (split > 1 ? 2u * (uint32_t)nt * kGmmRows * 4u : 0u);
}
GX_HD constexpr int gmm_stages(int ctas, int nt, int mode, int groups, int split) {
    const uint32_t n = (kGroupedSmem - kGroupedAlign - gmm_fixed_bytes(nt, mode, groups, split)) / gmm_stage_bytes(ctas, nt, mode);
    return n < (uint32_t)kGmmMaxStages ? (int)n : kGmmMaxStages;
}

// ------------------------------------------------------------- adapters

constexpr int kLoraRows = 32;                   // rows of a tile (MMA N)
constexpr int kLoraMaxStages = 12;
constexpr int kLoraEpiWarps = 4;
constexpr int kLoraThreads = 32 * (4 + kLoraEpiWarps);           // 8 warps: two CTAs of 128 registers a thread fit an SM
constexpr uint32_t kLoraHalfSm = 112u * 1024u;  // dynamic shared memory that leaves room for a second CTA
constexpr int kLoraSums = 6;                    // accumulators of h that take turns
constexpr uint32_t kLoraTmem = 256;             // columns: the sums of h, two tiles of results (32 each)
constexpr int kLoraK = 128;                     // elements of K per stage: two swizzled rows of 64
constexpr int kLoraSeg = 4;                     // stages that one accumulator of h sums where sums are long
static_assert((kLoraSums + 2) * kLoraRows <= kLoraTmem, "columns of TMEM");
constexpr uint32_t kLoraXTile = kLoraRows * 128u;
constexpr uint32_t kLoraStaging = kLoraEpiWarps * 16u * 32u * 4u;

// (ra: the pool's rank rounded up to 16, 32, 64 or 128)
GX_HD constexpr uint32_t lora_stage_bytes(int ra) { return 2u * (kLoraXTile + (uint32_t)ra * 128u); }
// B and h lie in blocks of up to 64 ranks, their rows swizzled over 32, 64 or
// 128 bytes: as many as the ranks fill
GX_HD constexpr uint32_t lora_blocks(int ra) { return ra > 64 ? 2u : 1u; }
GX_HD constexpr uint32_t lora_row(int ra) { return ra >= 64 ? 128u : (uint32_t)ra * 2u; }
GX_HD constexpr uint32_t lora_b_block(int ra) { return 128u * lora_row(ra); }
GX_HD constexpr uint32_t lora_h_block(int ra) { return (uint32_t)kLoraRows * lora_row(ra); }
GX_HD constexpr uint32_t lora_fixed_bytes(int ra, int groups) {
    return lora_blocks(ra) * (2u * lora_b_block(ra) + 3u * lora_h_block(ra)) + (uint32_t)kLoraRows * ra * 4u + kLoraStaging +
           kLoraRows * 4u + ((uint32_t)groups + 2u) * 4u;
}
// small ranks leave room for two CTAs per SM, whose phases overlap
GX_HD constexpr int lora_ctas_per_sm(int ra, int groups) {
    return kGroupedAlign + 2u * lora_stage_bytes(ra) + lora_fixed_bytes(ra, groups) <= kLoraHalfSm ? 2 : 1;
}
// stages of the ring: even, as two copying warps take them in turn. With 8192
// groups at rank 128 there is room for two, the fewest that work.
GX_HD constexpr int lora_stages(int ra, int groups) {
    const uint32_t have = lora_ctas_per_sm(ra, groups) == 2 ? kLoraHalfSm : kGroupedSmem;
    const uint32_t n = (have - kGroupedAlign - lora_fixed_bytes(ra, groups)) / lora_stage_bytes(ra);
    return (int)(n < (uint32_t)kLoraMaxStages ? n : kLoraMaxStages) & ~1;
}

}  // namespace gx
