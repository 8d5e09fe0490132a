// Tiles and shared memory of the products with 4-bit weights (plain C++, used
// by the kernels, by the entry points and by the host-side tests).
#pragma once

#include "gx_formats.h"

namespace gx {

constexpr int kQ4MaxIds = 256;                 // rows of a call that names each row's expert (one thread a row)
constexpr int kQ4Warps = 8;                    // they share K
constexpr int kQ4Threads = 32 * kQ4Warps;
constexpr int kQ4Stages = 3;

// Of NT tiles of eight columns (rows of x): tiles of 16 matrix rows per job,
// pairs of blocks per stage, bytes between the stage's rows (an odd number of 16
// bytes: eight rows then lie in different banks; 12 bytes more than the blocks
// take, as rows start on any 4 bytes)
GX_HD constexpr int q4_mt(int nt) { return nt == 1 ? 1 : 2; }
GX_HD constexpr int q4_pairs(int nt) { return nt == 1 ? 8 : 4; }
GX_HD constexpr int q4_pitch(bool q41, int nt) { return nt == 1 ? (q41 ? 336 : 304) : 176; }
GX_HD constexpr int q4_red_pitch(int nt) { return 16 * q4_mt(nt) + 4; }
// partial sums of the warps: two buffers where they are small
GX_HD constexpr int q4_buffers(int nt) { return nt == 1 ? 2 : 1; }
GX_HD constexpr uint32_t q4_smem(bool q41, int nt, int entries) {
    return (uint32_t)(kQ4Warps * kQ4Stages * 16 * q4_mt(nt) * q4_pitch(q41, nt)) +
           (uint32_t)(q4_buffers(nt) * kQ4Warps * 8 * nt * q4_red_pitch(nt) * 4) + (uint32_t)(entries + 1) * 4u;
}

}  // namespace gx
