"""Borders of groups that a device buffer may hold, in the products with 4-bit weights (host code, compiled for the test; the
kernel with such borders on the GPU)."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parent.parent / "galactus_b200" / "csrc"
CODE = """
#include "gx_q4_plan.h"
extern "C" int tiles(int lo, int hi, int n_rows, int least, int most, int cap) { return gx::q4_group_tiles(lo, hi, n_rows, least, most, cap); }
"""
LOW, HIGH = -2 ** 31, 2 ** 31 - 1


def test_tiles_of_any_borders(tmp_path):
    (tmp_path / "t.cpp").write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", str(CSRC), str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t.so")], check=True)
    tiles = C.CDLL(str(tmp_path / "t.so")).tiles
    edges = [LOW, LOW + 1, LOW + 23, -25, -1, 0, 1, 2, 23, 24, 25, 39, 40, 41, HIGH - 23, HIGH - 1, HIGH]
    for n_rows in (1, 24, 40, HIGH - 65536):
        for least, most in ((1, 24), (1, HIGH), (25, HIGH)):
            for lo in edges:
                for hi in edges:
                    n = hi - lo if 0 <= lo <= hi <= n_rows else 0
                    want = -(-n // 8) if least <= n <= most else 0
                    assert tiles(lo, hi, n_rows, least, most, 8) == want, (lo, hi, n_rows, least, most)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,size", [(2, 18), (3, 20)])
def test_wild_borders_among_many_groups(gxlib, dev, kind, size):
    """A thread looks at several groups together, some of them with borders whose difference is a small number in 32 bits."""
    torch = pytest.importorskip("torch")
    from test_gpu_q4 import check, error_code, want, weights
    rng = np.random.default_rng(1)
    E, K, N, P = 1600, 64, 20, 60
    w = weights(rng, E, N, K, kind)
    offsets = np.full(E + 1, -7, dtype=np.int32)
    e = np.full(P, -1)
    # groups of 5 rows, with borders in between that belong to no group
    for i in range(12):
        at = 130 * i + 3
        offsets[at], offsets[at + 1] = 5 * i, 5 * i + 5
        e[5 * i:5 * i + 5] = at
        offsets[at + 2:at + 5] = HIGH, LOW + 3, LOW
    x = torch.from_numpy(rng.standard_normal((P, K))).cuda().to(torch.float16)
    got = torch.full((P, N), 5.0, device="cuda")
    gxlib.mul_mat_q4(w, x, type=kind, offsets=torch.from_numpy(offsets).cuda(), out=got)
    assert error_code(gxlib) == 1
    check(got, *want(w, x, kind, e.tolist()))
