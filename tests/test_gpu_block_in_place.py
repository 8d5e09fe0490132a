"""Results of a block's end in place of what it reads, by every kernel that a shape may take."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# a warp, a CTA, a cluster a row, rings of rows (of eight and of sixteen warps), rows off 16 bytes
SIZES = [(50, 256), (40, 1000), (3, 20000), (700, 4096), (300, 8192), (60, 1001)]


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("what", ["residual", "y", "shared", "gate", "next over y"])
def test_in_place(gxlib, dev, T, H, what):
    rng = np.random.default_rng(T + H)
    rand = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()      # noqa: E731
    y, shared, gate, res, weight = rand(T, H), rand(T, H), rand(T, H), rand(T, H), rand(H)
    args = dict(shared=shared, norm=weight, gate=gate, residual=res, next_norm=weight, next_dtype=torch.float32)
    out, after = gxlib.block_out(y, **args)
    place = dict(residual=dict(out=res), y=dict(out=y), shared=dict(out=shared), gate=dict(out=gate))
    got, then = gxlib.block_out(y, **args, **(place[what] if what in place else dict(next_out=y)))
    assert torch.equal(got, out) and torch.equal(then, after)
    assert (got if what in place else then).data_ptr() in [t.data_ptr() for t in (y, shared, gate, res)]


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_in_place(gxlib, dev, T, H, dtype):
    rng = np.random.default_rng(T)
    x = torch.from_numpy(rng.standard_normal((T, H))).cuda().to(dtype)
    want = gxlib.rms_norm(x)
    assert gxlib.rms_norm(x, out=x) is x and torch.equal(x, want)
