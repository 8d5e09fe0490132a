"""Tiles and shared memory of the products with 4-bit weights, over every size
that the entry points accept (host code, compiled for the test)."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "galactus_b200" / "csrc"
CODE = """
#include "gx_grouped_plan.h"
#include "gx_q4_plan.h"
extern "C" {
void shape(int q41, long K, long n_rows, int * out) {
    const gx::Q4Shape s = gx::q4_shape(q41 != 0, K, n_rows);
    out[0] = s.warps; out[1] = s.cap; out[2] = s.buffers;
    out[3] = (int)gx::q4_smem(q41 != 0, K, s.warps, s.cap, s.buffers);
}
unsigned most() { return gx::kQ4Smem; }
int layout(int q41, int * out) {
    out[0] = gx::q4_pitch(q41 != 0); out[1] = gx::q4_stage_bytes(q41 != 0); out[2] = (int)gx::q4_pair_bytes(q41 != 0);
    out[3] = (int)gx::gmm_q4_pitch(q41 != 0); out[4] = (int)gx::gmm_q4_raw(q41 != 0);
    return gx::kQ4Pairs * 100 + gx::kGmmQ4Chunks;
}
int gmm_stages(int q41, int nt, int mode, int groups, int parts) { return gx::gmm_q4_stages(q41 != 0, nt, mode, groups, parts); }
unsigned gmm_smem(int q41, int nt, int mode, int groups, int parts) {
    return gx::kGroupedAlign + gx::gmm_q4_stages(q41 != 0, nt, mode, groups, parts) * gx::gmm_q4_stage_bytes(nt, parts) +
           gx::gmm_q4_fixed_bytes(q41 != 0, nt, mode, groups);
}
}
"""
MOST = 226 * 1024                 # dynamic shared memory of the grouped products' kernel


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    lib = C.CDLL(str(d / "plan.so"))
    lib.shape.argtypes = [C.c_int, C.c_long, C.c_long, C.POINTER(C.c_int)]
    return lib


@pytest.mark.parametrize("q41", [0, 1])
def test_few_rows_fit_for_every_length(plan, q41):
    """Warps come in fours (their rings in pairs), at least one row of x has room, and no tile is larger than what
    an mbarrier counts (2^20 - 1 bytes)."""
    out = (C.c_int * 4)()
    for K in range(64, 65536 + 64, 64):
        for rows in (1, 2, 7, 8, 9, 100000):
            plan.shape(q41, K, rows, out)
            warps, cap, buffers, smem = out
            assert warps in (4, 8, 12, 16) and 1 <= cap <= min(rows, 8) and buffers in (1, 2), (K, rows)
            assert smem <= plan.most() and cap * 2 * K < 1 << 20, (K, rows)


@pytest.mark.parametrize("q41", [0, 1])
def test_rows_of_a_stage(plan, q41):
    """A piece that starts on any 4 bytes of 16 fits its row; rows are an odd number of 16 bytes apart; stages, and the
    two halves of gated ones, start on 128 bytes, as boxes need; a stage's boxes start on 16 bytes."""
    out = (C.c_int * 5)()
    code = plan.layout(q41, out)
    pair = 40 if q41 else 36
    for pitch, pairs in ((out[0], code // 100), (out[3], code % 100)):
        assert pitch >= pairs * pair + 12 and pitch % 16 == 0 and pitch // 16 % 2 == 1 and pitch // 4 <= 256
        assert pairs * pair % 16 == 0 and 32 * pitch % 128 == 0 and 16 * pitch % 128 == 0
    assert out[1] == 32 * out[0] and out[2] % 16 == 0 and out[4] % (32 * out[3]) == 0


@pytest.mark.parametrize("q41", [0, 1])
@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("first,parts", [(160, 2), (256, 2), (160, 3), (256, 3)])
def test_many_rows_ring(plan, q41, mode, first, parts):
    """Two stages at least for every number of matrices, with tiles of 32 rows or more."""
    for groups in range(1, 8193):
        nt = first
        while plan.gmm_stages(q41, nt, mode, groups, parts) < 2:
            nt -= 32
            assert nt >= 32, groups
        assert plan.gmm_smem(q41, nt, mode, groups, parts) <= MOST, groups
