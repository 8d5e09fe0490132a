// Tiles and shared memory of the products with 4-bit weights (plain C++, used
// by the kernels, by the entry points and by the host-side tests).
#pragma once

#include "gx_formats.h"

namespace gx {

constexpr int kQ4MaxIds = 256;                 // rows of a call that names each row's expert (one thread a row)

constexpr int kQ4Warps = 16;                   // of a CTA, at most
constexpr int kQ4Stages = 2;                   // of the ring that two warps share
constexpr int kQ4Pairs = 8;                    // pairs of blocks per stage
constexpr int kQ4Mt = 2;                       // 16-row tiles of the matrix per job
constexpr int kQ4Cols = 8;                     // rows of x per job
// Bytes between the rows of a stage: an odd number of 16 bytes (eight rows then
// lie in different banks), 12 more than the blocks take (rows start on any 4 bytes)
GX_HD constexpr int q4_pitch(bool q41) { return 16 * (((kQ4Pairs * (q41 ? 40 : 36) + 12 + 15) / 16) | 1); }
GX_HD constexpr int q4_stage_bytes(bool q41) { return 16 * kQ4Mt * q4_pitch(q41); }
// A warp's sums: [columns][kQ4Red]
constexpr int kQ4Red = 16 * kQ4Mt + 4;
// two warps: their ring and their sums
GX_HD constexpr uint32_t q4_pair_bytes(bool q41) { return (uint32_t)(kQ4Stages * q4_stage_bytes(q41) + 2 * kQ4Cols * kQ4Red * 4); }
// a row of x (the 32 bytes more put four rows into different banks)
GX_HD constexpr int64_t q4_x_pitch(int64_t K) { return 2 * K + 32; }
// dynamic shared memory; the lists that the kernel declares itself take 8 KB
constexpr uint32_t kQ4Smem = (227u - 8u) * 1024u;

struct Q4Shape {
    int warps, cap, buffers;                   // warps of a CTA, rows of x per tile, tiles of x at once
};
// As many warps as leave room for two tiles of x (or one; or fewer rows, which
// only very long rows need)
inline Q4Shape q4_shape(bool q41, int64_t K, int64_t n_rows) {
    const int64_t row = q4_x_pitch(K);
    const int cols = n_rows < kQ4Cols ? (int)n_rows : kQ4Cols;
    for (int w = kQ4Warps; w >= 4; w -= 4)
        for (int b = 2; b >= 1; --b)
            if (w / 2 * (int64_t)q4_pair_bytes(q41) + b * cols * row <= kQ4Smem) return {w, cols, b};
    const int64_t room = (int64_t)kQ4Smem - 2 * (int64_t)q4_pair_bytes(q41);
    return {4, (int)(room / row), 1};
}
GX_HD constexpr uint32_t q4_smem(bool q41, int64_t K, int warps, int cap, int buffers) {
    return (uint32_t)(warps / 2) * q4_pair_bytes(q41) + (uint32_t)(buffers * cap * q4_x_pitch(K));
}

// Tiles of `cap` rows in the group of rows [lo, hi), if it has from `least` (>= 1) to
// `most` rows. Borders that do not ascend or leave the rows, whatever they hold (their
// difference may pass 32 bits), are those of no rows.
GX_HD int q4_group_tiles(int lo, int hi, int n_rows, int least, int most, int cap) {
    if (lo < 0 || hi < lo || hi > n_rows) return 0;
    const int n = hi - lo;
    return n < least || n > most ? 0 : (n - 1) / cap + 1;
}

}  // namespace gx
