"""Infinities and NaN in rows that are kept: they stay in their row, and in their element where nothing takes the row's norm."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
# a warp, a CTA, a cluster a row, rings of rows, and rows off 16 bytes
SIZES = [(50, 2, 256), (40, 2, 1000), (3, 2, 20000), (300, 2, 4096), (60, 2, 1001), (60, 40, 136)]


@pytest.mark.parametrize("T,k,H", SIZES)
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("norm", [False, True])
def test_bad_element(gxlib, dev, T, k, H, bad, norm):
    rng = np.random.default_rng(H)
    rand = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()      # noqa: E731
    y, w, res = rand(T, k, H), 0.5 + rand(T, k).abs(), rand(T, H)
    weight = 0.5 + rand(H).abs()
    args = dict(weights=w, residual=res, norm=weight if norm else None, next_norm=weight, next_dtype=torch.float32)
    out, after = (t.clone() for t in gxlib.block_out(y, **args))
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(after).all())
    row, at = T // 2, H - 3
    y[row, k - 1, at] = bad
    got, then = gxlib.block_out(y, **args)
    others = torch.arange(T, device="cuda") != row
    assert torch.equal(got[others], out[others]) and torch.equal(then[others], after[others])
    rest = torch.arange(H, device="cuda") != at
    if norm or bad != bad:
        # inf / sqrt(inf) at its element, 0 elsewhere (the residual is left); a NaN takes the whole row with it
        assert bool(torch.isnan(got[row, at]))
        if norm:
            assert bool(torch.isnan(got[row, rest]).all()) if bad != bad else torch.equal(got[row, rest], res[row, rest])
        else:
            assert torch.equal(got[row, rest], out[row, rest])
        assert bool(torch.isnan(then[row]).all())
    else:
        assert float(got[row, at]) == bad and torch.equal(got[row, rest], out[row, rest])
        assert bool(torch.isnan(then[row, at])) and bool((then[row, rest] == 0).all())
    x = res.clone()
    x[row, at] = bad
    normed = gxlib.rms_norm(x, weight)
    assert torch.equal(normed[others], gxlib.rms_norm(res, weight)[others]) and bool(torch.isnan(normed[row, at]))
    assert bool(torch.isnan(normed[row, rest]).all()) if bad != bad else bool((normed[row, rest] == 0).all())
