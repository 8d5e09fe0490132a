"""Matrix tiles of 4-bit weights whose rows do not start on 16 bytes: the last row's last bytes are moved by hand."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_q4 import BF16, F32, Q4_0, Q4_1, check, error_code, want, weights  # noqa: E402


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("K", [64, 128, 192, 320, 448, 1600])
@pytest.mark.parametrize("N", [1, 33, 128, 150])
def test_last_row(gxlib, dev, kind, K, N):
    """The matrices at the very end of their memory, against the same ones with rows on 16 bytes (copied as boxes): the arithmetic
    is the same, and so are the bits."""
    rng = np.random.default_rng(K + N)
    G, P = 2, 80
    w = weights(rng, G, N, K, kind)
    rb = w.shape[2]
    wide = torch.zeros((G, N, (rb + 15) // 16 * 16), dtype=torch.uint8, device="cuda")
    wide[:, :, :rb] = w
    x = torch.from_numpy(rng.standard_normal((P, K))).cuda().to(BF16)
    offsets = torch.tensor([0, 30, P], dtype=torch.int32, device="cuda")
    aligned = gxlib.mul_mat_q4(wide[:, :, :rb], x, type=kind, offsets=offsets, out_dtype=F32)
    check(aligned, *want(w, x, kind, [0] * 30 + [1] * 50))
    both = gxlib.mul_mat_q4_glu(wide[:, :, :rb], wide.flip(0)[:, :, :rb], x, type=kind, offsets=offsets)
    for _ in range(20):
        assert torch.equal(gxlib.mul_mat_q4(w, x, type=kind, offsets=offsets, out_dtype=F32), aligned)
        assert torch.equal(gxlib.mul_mat_q4_glu(w, w.flip(0), x, type=kind, offsets=offsets), both)
    assert error_code(gxlib) == 0
