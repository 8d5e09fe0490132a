"""Waits that run out inside the kernels (products with 4-bit weights, rings of rows): what is written is the right value or
NaN, never a sum of what was not there."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_q4 import BF16, F16, F32, Q4_0, Q4_1, weights  # noqa: E402

ROOT = Path(__file__).resolve().parent
TIMEOUT = 2


@pytest.fixture(scope="module")
def late(gxlib, dev):
    """The kernels with a wait that can be made to run out: a library of its own, built beside the test."""
    from galactus_b200 import build as b
    src, out = ROOT / "native" / "late_waits.cu", ROOT / "_build" / "late_waits.so"
    deps = [src, Path(b.__file__), ROOT.parent / "include" / "galactus_b200.h"] + [b.CSRC / f for f in b.SOURCES + b.HEADERS]
    if not out.exists() or any(d.stat().st_mtime > out.stat().st_mtime for d in deps):
        out.parent.mkdir(exist_ok=True)
        subprocess.run([b.nvcc(), *b.NVCC_FLAGS, "-shared", "-Xlinker", "-Bsymbolic", "-I", str(b.CSRC), "-I", str(ROOT.parent / "include"),
                        str(src), "-o", str(out)], check=True)
    lib = C.CDLL(str(out))
    for name in ("gx_mul_mat_q4", "gx_mul_mat_q4_glu", "gx_block_out"):
        f = getattr(lib, name)
        f.restype, f.argtypes = gxlib._lib._SIGS[name]
    return lib


def run(late, call, out, block, warp, at):
    """(results, waits of that warp)"""
    out.fill_(3.0)
    assert late.late_set(block, warp, at) == 0
    assert call() == 0
    torch.cuda.synchronize()
    assert late.late_error() == (TIMEOUT if at >= 0 else 0)
    return out.clone(), late.late_seen()


def points(n):
    return sorted({0, 1, n // 2, n - 2, n - 1} & set(range(n)))


def check(late, call, out, blocks, warps):
    """Waits of the warps in turn: results are the right bits or NaN, and there is NaN where nothing came after the first."""
    good, _ = run(late, call, out, -1, -1, -1)
    assert bool(torch.isfinite(good).all())
    tried = 0
    for block in blocks:
        for warp in warps:
            same, n = run(late, call, out, block, warp, -1)
            assert torch.equal(same, good)
            tried += n > 0                                                # (a block without jobs waits for nothing)
            for at in points(n):
                got, _ = run(late, call, out, block, warp, at)
                nan = torch.isnan(got)
                assert bool((nan | (got == good)).all()), (block, warp, at)
                assert at > 0 or bool(nan.any()), (block, warp)
    assert tried >= len(warps)
    again, _ = run(late, call, out, -1, -1, -1)
    assert torch.equal(again, good)


def q4_args(w, x, kind, ids, n_rows, gather, out):
    G, N, nb = w.shape
    return (kind, w.data_ptr(), x.shape[1], N, nb, N * nb, G, 30 if x.dtype == BF16 else 1, x.data_ptr(), x.shape[0], 2 * x.shape[1],
            ids.data_ptr() if ids is not None else None, None, None, n_rows, gather, 0, 0 if out.dtype == F32 else 1, out.data_ptr(),
            N * out.element_size(), torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("kind,dtype", [(Q4_0, BF16), (Q4_1, F16)])
@pytest.mark.parametrize("K,N,E,rows", [(4096, 64, 1, 4), (1024, 2000, 40, 120), (2048, 320, 3, 100)])
def test_streamed_products(late, kind, dtype, K, N, E, rows):
    """Few jobs shared by a CTA's warps, and many with several tiles of rows (rows of blocks on 16 bytes: copied as boxes, by the
    first warp of each two, while warp 0 also copies the rows of x)."""
    rng = np.random.default_rng(K)
    w = weights(rng, E, N, K, kind)
    x = torch.from_numpy(rng.standard_normal((rows, K))).cuda().to(dtype)
    ids = torch.from_numpy(rng.integers(0, E, rows).astype(np.int32)).cuda()
    out = torch.empty((rows, N), dtype=F32, device="cuda")
    args = q4_args(w, x, kind, ids, rows, 1, out)
    check(late, lambda: late.gx_mul_mat_q4(*args), out, [0, 1, 2], [0, 1, 2, 5])


@pytest.mark.parametrize("parts", ["plain", "norm", "next", "all"])
@pytest.mark.parametrize("T,k,H", [(700, 2, 4096), (300, 3, 8192)])
def test_rings_of_rows(gxlib, late, parts, T, k, H):
    """One warp of eight (or sixteen) that compute, with each of the sums over the row there or not, and the warp that copies."""
    rng = np.random.default_rng(H)
    rand = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()      # noqa: E731
    y, weights_, res, norm, after = rand(T, k, H), rand(T, k), rand(T, H), rand(H), rand(H)
    both = torch.empty((2, T, H), device="cuda")
    d = gxlib._lib.gx_block_desc()
    d.ne0, d.ne1, d.k, d.scale, d.eps, d.next_eps = H, T, k, 1.0, 1e-6, 1e-6
    d.y, d.nby1, d.nby2, d.weights = y.data_ptr(), 4 * H, 4 * H * k, weights_.data_ptr()
    d.residual, d.nbr, d.dst, d.nbd = res.data_ptr(), 4 * H, both.data_ptr(), 4 * H
    if parts in ("norm", "all"):
        d.norm = norm.data_ptr()
    if parts in ("next", "all"):
        d.next, d.nbn, d.next_norm = both.data_ptr() + 4 * T * H, 4 * H, after.data_ptr()
    else:
        both = both[:1]
    out = both.view(-1, H)
    check(late, lambda: late.gx_block_out(C.byref(d), torch.cuda.current_stream().cuda_stream), out, [0, 17], [0, 3, H // 512])
    if parts in ("norm", "all"):
        # the last expert's row of a block's last token: its warp's share of the norm is lost to the whole row
        _, n = run(late, lambda: late.gx_block_out(C.byref(d), torch.cuda.current_stream().cuda_stream), out, 17, 3, -1)
        got, _ = run(late, lambda: late.gx_block_out(C.byref(d), torch.cuda.current_stream().cuda_stream), out, 17, 3, n - 2)
        bad = torch.isnan(got).sum(1)
        assert set(bad.tolist()) == {0, H} and int((bad == H).sum()) == both.shape[0]


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("scatter", [False, True])
def test_tiles_of_many_rows(late, kind, glu, dtype, scatter):
    """The warps that read the accumulators, at their last wait (all else has then ended): their share of the last tile is NaN, and
    nothing keeps what dst held before."""
    rng = np.random.default_rng(5)
    E, N, K, P = 3, 300, 512, 700
    w, up = weights(rng, E, N, K, kind), weights(rng, E, N, K, kind)
    x = torch.from_numpy(rng.standard_normal((P, K))).cuda().to(F16)
    offsets = torch.tensor([0, 200, 430, P], dtype=torch.int32, device="cuda")
    order = torch.from_numpy(rng.permutation(P).astype(np.int32)).cuda()
    out = torch.empty((P, N), dtype=dtype, device="cuda")
    head = (kind, w.data_ptr(), up.data_ptr()) if glu else (kind, w.data_ptr())
    args = head + (K, N, w.shape[2], N * w.shape[2], E, 1, x.data_ptr(), P, 2 * K, None, offsets.data_ptr(), order.data_ptr(), P, 1, int(scatter))
    args += ((0, 0.0, 0.0) if glu else ()) + (0 if dtype == F32 else 1, out.data_ptr(), N * out.element_size())
    f = late.gx_mul_mat_q4_glu if glu else late.gx_mul_mat_q4
    call = lambda: f(*args, torch.cuda.current_stream().cuda_stream)                           # noqa: E731
    good, _ = run(late, call, out, -1, -1, -1)
    tried = 0
    for block in (0, 1, 6):
        for warp in range(4, 8):
            same, n = run(late, call, out, block, warp, -1)
            assert torch.equal(same, good)
            if n:
                got, _ = run(late, call, out, block, warp, n - 1)
                nan = torch.isnan(got)
                assert bool((nan | (got == good)).all()), (block, warp)
                tried += int(nan.any())
    assert tried >= 8
