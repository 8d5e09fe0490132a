"""Products of few rows with 4-bit weights: rows with a mean beside their deviation, where the sums of a block's codes are small
beside the sums of its elements."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_q4 import BF16, BLOCK, F16, F32, Q4_0, Q4_1, weights  # noqa: E402


def centred(rng, N, K, kind):
    """(blocks, d, m, codes): Q4_1 minima near -7.5 d, as weights around zero have them."""
    w = weights(rng, 1, N, K, kind)
    b = w.cpu().numpy().reshape(N, K // 32, BLOCK[kind])
    d = np.ascontiguousarray(b[..., 0:2]).view(np.float16)
    m = np.zeros_like(d)
    if kind == Q4_1:
        m = (-d.astype(np.float32) * (6.5 + 2.0 * rng.random(d.shape))).astype(np.float16)
        b[..., 2:4] = m.view(np.uint8)
    qs = b[..., BLOCK[kind] - 16:]
    q = np.concatenate([qs & 15, qs >> 4], axis=-1)
    as64 = lambda a: torch.from_numpy(a.astype(np.float64)).cuda()      # noqa: E731
    return torch.from_numpy(b.reshape(1, N, -1)).cuda(), as64(d[..., 0]), as64(m[..., 0]), as64(q)


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("mean", [0.0, 0.5, 1.0, 3.0])
@pytest.mark.parametrize("K", [256, 1024, 7168])
def test_rows_with_a_mean(gxlib, dev, kind, dtype, mean, K):
    """The error on the whole. A product of a code and an element has 15 bits, so what the tensor cores cut off a sum of 16 of them is
    a step (2^-23) of the sum, and of the largest product for those 2^9 times smaller. The sums are those of the first 16 and of all
    32 elements of a block: of (q - 8) x, with those of x beside them (F16), or of (16 + q) x that begin with -24 or -16 times the
    sum of x (BF16). The blocks' parts are added in f32, half a step of the sum so far at each of one or two fmas. Errors of blocks
    have signs of their own: their squares add."""
    rng = np.random.default_rng(K + int(8 * mean))
    N, R = 96, 8
    w, d, m, q = centred(rng, N, K, kind)
    x = torch.from_numpy(mean + rng.standard_normal((R, K))).cuda().to(dtype)
    got = gxlib.mul_mat_q4(w, x, type=kind, out_dtype=F32).double()

    x64 = x.double().view(R, K // 32, 2, 16)
    low, all_ = 8.0 if kind == Q4_0 else 0.0, x64.sum((2, 3))
    half = lambda c: torch.einsum("rbhi,nbhi->rnbh", x64, c.view(N, K // 32, 2, 16)).cumsum(-1)      # noqa: E731
    y = (d * half(q - low)[..., 1] + m * all_[:, None]).cumsum(-1)
    sums = x64.sum(3).cumsum(-1)[:, None]                                  # [R, 1, blocks, 2]
    largest = x64.abs().amax((2, 3))[:, None]
    if dtype == F16:
        cut = half(q - 8.0).abs().sum(-1) + 2 * 8.0 * largest
        off = (d * cut) ** 2
        if kind == Q4_1:
            off = off + ((m + 8.0 * d) * (sums.abs().sum(-1) + 2 * largest)) ** 2
    else:
        take = 24.0 if kind == Q4_0 else 16.0
        cut = take * sums.abs().sum(-1) + (half(q + 16.0) - take * sums[..., 1:]).abs().sum(-1) + 2 * (take + 31.0) * largest
        off = (d * cut) ** 2
        if kind == Q4_1:
            off = off + (m * sums.abs().sum(-1)) ** 2
    adds = (1 if kind == Q4_0 else 2) * (y ** 2).sum(-1)
    bound = (off.sum(-1) * 2.0 ** -46 + adds * 2.0 ** -48).mean().sqrt()
    assert float((got - y[..., -1]).square().mean().sqrt()) <= float(bound)


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("rows", [8, 24, 25, 80])
def test_weights_at_the_border_of_the_rows_type(gxlib, dev, kind, rows):
    """F16 rows: the largest weights, 65504 and a little less, on both sides of the length from which tiles of weights are made. (d is
    8188: every weight is a multiple of 4 of at most 15 bits, and so is its product with an element of -1, 0 or 1.)"""
    rng = np.random.default_rng(rows)
    N, K = 40, 128
    w, _, _, q = centred(rng, N, K, kind)
    b = w.cpu().numpy().reshape(N, K // 32, BLOCK[kind])
    b[..., 0:2] = np.frombuffer(np.float16(8188.0).tobytes(), np.uint8)
    if kind == Q4_1:
        b[..., 2:4] = np.frombuffer(np.float16(-65504.0).tobytes(), np.uint8)
    x = torch.from_numpy(rng.integers(-1, 2, (rows, K)).astype(np.float16)).cuda()
    want = x.double() @ (8188.0 * (q - 8.0)).view(N, K).T
    got = gxlib.mul_mat_q4(torch.from_numpy(b.reshape(1, N, -1)).cuda(), x, type=kind, out_dtype=F32)
    # (whole numbers below 2^24 after a division by 4)
    assert torch.equal(got.double(), want)
