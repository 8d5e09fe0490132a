"""Tiles and shared memory of the kernels on grouped rows, over every size that
the entry points accept (host code, compiled for the test)."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "galactus_b200" / "csrc"
CODE = """
#include "gx_grouped_plan.h"
extern "C" {
int lora_stages(int ra, int groups) { return gx::lora_stages(ra, groups); }
unsigned lora_smem(int ra, int groups) {
    return gx::kGroupedAlign + gx::lora_stages(ra, groups) * gx::lora_stage_bytes(ra) + gx::lora_fixed_bytes(ra, groups);
}
int lora_per_sm(int ra, int groups) { return gx::lora_ctas_per_sm(ra, groups); }
int gmm_stages(int ctas, int nt, int mode, int groups, int split) { return gx::gmm_stages(ctas, nt, mode, groups, split); }
unsigned gmm_smem(int ctas, int nt, int mode, int groups, int split) {
    return gx::kGroupedAlign + gx::gmm_stages(ctas, nt, mode, groups, split) * gx::gmm_stage_bytes(ctas, nt, mode) +
           gx::gmm_fixed_bytes(nt, mode, groups, split);
}
}
"""
MOST = 227 * 1024 - 1024          # what a CTA may have, less what the kernels declare themselves
GROUPS = sorted({1, 2, 100, 1024, 4096, *range(8000, 8193)})


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(CODE)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    return C.CDLL(str(d / "plan.so"))


@pytest.mark.parametrize("ra", [16, 32, 64, 128])
def test_adapters_ring_has_two_stages_for_every_group_count(plan, ra):
    """Two copying warps take the stages in turn: an even number of them, two at least."""
    for g in range(1, 8193):
        n = plan.lora_stages(ra, g)
        assert n >= 2 and n % 2 == 0, (ra, g, n)
        assert plan.lora_smem(ra, g) <= (112 * 1024 if plan.lora_per_sm(ra, g) == 2 else MOST), (ra, g)


@pytest.mark.parametrize("mode,ctas,nt,split", [(0, 1, 32, s) for s in (1, 2, 4, 8)] + [(1, 1, 32, s) for s in (1, 2, 4, 8)] +
                         [(m, 1, nt, 1) for m in (0, 1) for nt in (64, 128)] + [(m, 2, nt, 1) for m in (0, 1) for nt in (160, 256)] +
                         [(2, 2, 256, 1)])
def test_products_ring(plan, mode, ctas, nt, split):
    for g in GROUPS:
        assert plan.gmm_stages(ctas, nt, mode, g, split) >= 2 and plan.gmm_smem(ctas, nt, mode, g, split) <= MOST, g


def test_types_that_are_not_quantised(gxlib):
    """Their activations have their own type (gx_quantize_rows' argument), their rows two or four bytes an element."""
    for t, size in ((gxlib.TYPE_F32, 4), (gxlib.TYPE_F16, 2), (gxlib.TYPE_BF16, 2)):
        assert gxlib.vec_dot_type(t) == t and gxlib.row_bytes(t, 129) == 129 * size
    assert gxlib.vec_dot_type(gxlib.TYPE_Q8_0) == gxlib.vec_dot_type(gxlib.TYPE_MXFP4) == gxlib.TYPE_Q8_0
    assert gxlib.vec_dot_type(gxlib.TYPE_Q4_K) == gxlib.vec_dot_type(gxlib.TYPE_IQ1_S) == gxlib.TYPE_Q8_K
