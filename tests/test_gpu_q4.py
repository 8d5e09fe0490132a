"""Products with 4-bit weights on the GPU against the formula in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

Q4_0, Q4_1 = 2, 3
BLOCK = {Q4_0: 18, Q4_1: 20}
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ALPHA, LIMIT = 1.702, 7.0


def weights(rng, G, N, K, kind):
    """Random blocks: codes of every value, scales of either sign."""
    nb = K // 32
    b = rng.integers(0, 256, (G, N, nb, BLOCK[kind]), dtype=np.uint8)
    d = (0.004 * (0.5 + rng.random((G, N, nb, 1))) * rng.choice([-1.0, 1.0], (G, N, nb, 1))).astype(np.float16)
    b[..., 0:2] = d.view(np.uint8)
    if kind == Q4_1:
        b[..., 2:4] = (0.03 * rng.standard_normal((G, N, nb, 1))).astype(np.float16).view(np.uint8)
    return torch.from_numpy(b.reshape(G, N, nb * BLOCK[kind])).cuda()


def parts(w, kind):
    """(weights, per element the largest code times |d| plus what is taken off, times |d|) in 64 bits."""
    b = w.cpu().numpy().reshape(*w.shape[:-1], -1, BLOCK[kind])
    d = np.ascontiguousarray(b[..., 0:2]).view(np.float16).astype(np.float64)
    qs = b[..., BLOCK[kind] - 16:]
    q = np.concatenate([qs & 15, qs >> 4], axis=-1).astype(np.float64)
    if kind == Q4_0:
        v, a = d * (q - 8.0), np.abs(d) * 55.0 + 0.0 * q       # (16 + q, and 24 taken off)
    else:
        m = np.ascontiguousarray(b[..., 2:4]).view(np.float16).astype(np.float64)
        v, a = d * q + m, np.abs(d) * 47.0 + np.abs(m) + 0.0 * q
    return tuple(torch.from_numpy(t.reshape(*w.shape[:-1], -1)).cuda() for t in (v, a))


def want(w, x, kind, e, out=F32):
    """Row j of x times matrix e[j] (-1: none) in 64 bits, and how far f32 sums may be off: the tensor cores add a block's
    64 products of codes (at most 31 |d x|, and 24 |d x| taken off; F16 64 + q and 72, of which as much is left) within 6e-9 of
    their magnitudes each, then the block's sums are added in f32, K / 32 roundings of half a step. In calls of many rows a Q4_1
    weight is taken to 22 bits (F16 rows), or to 24 or 16 (BF16 rows; f32 results, others): off by half of the last."""
    n = w.shape[1]
    y = torch.zeros((len(e), n), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(y)
    K = x.shape[1]
    cut = 0.0 if kind == Q4_0 else 2.0 ** -22 if x.dtype == F16 else 2.0 ** -24 if out == F32 else 2.0 ** -16
    for g in sorted(set(int(v) for v in e if v >= 0)):
        rows = torch.tensor([j for j, v in enumerate(e) if v == g], device="cuda")
        v, a = parts(w[g], kind)
        xs = x[rows].double()
        y[rows] = xs @ v.T
        tol[rows] = (xs.abs() @ a.T) * 64 * 6e-9 + (xs.abs() @ v.abs().T) * ((K // 32 + 8) * 2.0 ** -24 + cut)
    return y, tol


def want_glu(gate, up, x, kind, e, act, out=F32):
    g, eg = want(gate, x, kind, e, out)
    u, eu = want(up, x, kind, e, out)
    if act:
        ok = g < LIMIT
        g, eg = g.clamp(max=LIMIT), torch.where(ok | ((g - LIMIT).abs() < eg), eg, 0.0)
        u = u.clamp(-LIMIT, LIMIT) + 1.0
        s = torch.sigmoid(ALPHA * g)
    else:
        s = torch.sigmoid(g)
    y = g * s * u
    # |d(x sigmoid(a x))/dx| <= 1.1; the exp is |x| + 2 steps of f32 off, the quotient two
    return y, 1.1 * eg * u.abs() + (g * s).abs() * eu + 1.1 * eg * eu + y.abs() * (g.abs() * 2 + 8) * 2.0 ** -23


def check(got, y, tol, skip=None, rms=6 * 4 * 2.0 ** -23):
    assert got.shape == y.shape
    half = 0.0 if got.dtype == F32 else torch.finfo(got.dtype).eps / 2
    tiny = 0.0 if got.dtype == F32 else torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bad = (got.double() - y).abs() > tol * (1 + half) + half * y.abs() + tiny
    if skip is not None:
        bad[skip] = False
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, at {bad.nonzero()[:4].tolist()}"
    if got.dtype == F32 and y.numel() >= 64 and rms is not None:
        # and on the whole: a block's sums are at most 6 times its result (16 + q and 24 beside q - 8), cut by a step of f32 in
        # each of four products of 16 elements
        keep = torch.ones(len(y), dtype=torch.bool, device=y.device)
        if skip is not None:
            keep[skip] = False
        assert float((got[keep].double() - y[keep]).norm()) <= rms * float(y[keep].norm())


def error_code(gxlib):
    import ctypes as C
    c = C.c_int32()
    gxlib.check(gxlib.lib().gx_device_error(C.byref(c)))
    return c.value


SIZES = [(64, 1), (64, 7), (128, 16), (192, 33), (704, 130), (1024, 64), (2880, 45), (4096, 24), (7168, 17)]


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("K,N", SIZES)
def test_dense(gxlib, dev, kind, dtype, out, K, N):
    rng = np.random.default_rng(K + N)
    w = weights(rng, 1, N, K, kind)
    for rows in (1, 2, 8, 9, 17, 31, 32, 33, 70):
        x = torch.from_numpy(rng.standard_normal((rows, K))).cuda().to(dtype)
        got = gxlib.mul_mat_q4(w, x, type=kind, out_dtype=out)
        check(got, *want(w, x, kind, [0] * rows, out))
    assert error_code(gxlib) == 0


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F16)])
@pytest.mark.parametrize("T,k,E,K,N", [(1, 8, 128, 768, 96), (1, 1, 1, 64, 3), (3, 4, 8, 320, 50), (19, 8, 64, 128, 40), (64, 4, 3, 256, 33),
                                       (256, 1, 200, 64, 16)])
def test_ids(gxlib, dev, kind, dtype, out, T, k, E, K, N):
    rng = np.random.default_rng(T * k + E)
    w = weights(rng, E, N, K, kind)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    ids[rng.random((T, k)) < 0.2] = -1
    dids = torch.from_numpy(ids).cuda()
    flat = ids.reshape(-1).tolist()
    none = torch.tensor([j for j, v in enumerate(flat) if v < 0], dtype=torch.long, device="cuda")
    # one row of x per token, then one per pair
    x = torch.from_numpy(rng.standard_normal((T, K))).cuda().to(dtype)
    keep = torch.full((T * k, N), 7.0, dtype=out, device="cuda")
    got = gxlib.mul_mat_q4(w, x, type=kind, ids=dids, gather=k, out=keep)
    y, tol = want(w, x.repeat_interleave(k, 0), kind, flat)
    check(got, y, tol, none)
    assert bool((got[none] == 7.0).all())
    x = torch.from_numpy(rng.standard_normal((T * k, K))).cuda().to(dtype)
    for gather in (0, 1):
        got = gxlib.mul_mat_q4(w, x, type=kind, ids=dids, gather=gather, out_dtype=out)
        check(got, *want(w, x, kind, flat), none)
    assert error_code(gxlib) == 0


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("T,k,E,K,N", [(5, 2, 8, 64, 20), (64, 8, 128, 128, 33), (300, 4, 16, 256, 70), (1031, 8, 64, 192, 40),
                                       (40, 1, 8192, 64, 16), (700, 2, 3, 320, 130)])
def test_groups(gxlib, dev, kind, dtype, out, T, k, E, K, N):
    rng = np.random.default_rng(T + E)
    w = weights(rng, E, N, K, kind) if E < 8192 else weights(rng, 16, N, K, kind).repeat(512, 1, 1)
    ids = np.minimum(rng.zipf(1.4, (T, k)) - 1, E - 1).astype(np.int32)
    ids[rng.random((T, k)) < 0.1] = -1
    order, offsets = gxlib.group_rows(torch.from_numpy(ids).cuda(), E)
    flat = ids.reshape(-1).tolist()
    n = int(offsets[-1])
    x = torch.from_numpy(rng.standard_normal((T, K))).cuda().to(dtype)
    none = torch.tensor([j for j, v in enumerate(flat) if v < 0], dtype=torch.long, device="cuda")
    keep = torch.full((T * k, N), 7.0, dtype=out, device="cuda")
    got = gxlib.mul_mat_q4(w, x, type=kind, offsets=offsets, order=order, gather=k, scatter=True, out=keep)
    y, tol = want(w, x.repeat_interleave(k, 0), kind, flat, out)
    check(got, y, tol, none)
    assert bool((got[none] == 7.0).all())
    # into expert order, and from expert order
    at = order.long()[:n]
    h = gxlib.mul_mat_q4(w, x, type=kind, offsets=offsets, order=order, gather=k, out_dtype=out)
    check(h[:n], y[at], tol[at])
    xs = x.repeat_interleave(k, 0)[order.long()].contiguous()
    got = gxlib.mul_mat_q4(w, xs, type=kind, offsets=offsets, order=order, scatter=True, out_dtype=out)
    check(got, y, tol, none)
    got = gxlib.mul_mat_q4(w, xs, type=kind, offsets=offsets, out_dtype=out)
    check(got[:n], y[at], tol[at])
    assert error_code(gxlib) == 0


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("T,k,E,K,N", [(1, 4, 16, 2880, 90), (1, 8, 8, 64, 1), (3, 8, 64, 512, 45), (200, 4, 16, 128, 60)])
def test_glu(gxlib, dev, kind, act, dtype, out, T, k, E, K, N):
    rng = np.random.default_rng(T + K + act)
    gate, up = weights(rng, E, N, K, kind), weights(rng, E, N, K, kind)
    ids = np.stack([rng.choice(E, k, replace=False) for _ in range(T)]).astype(np.int32)
    x = torch.from_numpy(3.0 * rng.standard_normal((T, K))).cuda().to(dtype)
    flat = ids.reshape(-1).tolist()
    y, tol = want_glu(gate, up, x.repeat_interleave(k, 0), kind, flat, act, out)
    dids = torch.from_numpy(ids).cuda()
    if T * k <= 256:
        check(gxlib.mul_mat_q4_glu(gate, up, x, type=kind, ids=dids, gather=k, act=act, out_dtype=out), y, tol)
    order, offsets = gxlib.group_rows(dids, E)
    check(gxlib.mul_mat_q4_glu(gate, up, x, type=kind, offsets=offsets, order=order, gather=k, scatter=True, act=act, out_dtype=out), y, tol)
    assert error_code(gxlib) == 0


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("pad", [4, 8, 12, 20, 64])
def test_strides(gxlib, dev, kind, pad):
    """Rows and matrices on every offset inside 16 bytes, rows of x and of the result further apart, a result with guard columns."""
    rng = np.random.default_rng(pad)
    G, N, K, T = 3, 21, 192, 11
    w = weights(rng, G, N, K, kind)
    rb = w.shape[2]
    wide = torch.zeros(G * (N * (rb + pad) + 4 * pad) + 64, dtype=torch.uint8, device="cuda")
    view = wide.as_strided((G, N, rb), (N * (rb + pad) + 4 * pad, rb + pad, 1))
    view.copy_(w)
    x = torch.from_numpy(rng.standard_normal((T, K + 24))).cuda().to(BF16)[:, :K]
    out = torch.full((T, N + 5), 3.0, dtype=F32, device="cuda")
    e = rng.integers(0, G, T).astype(np.int32)
    gxlib.mul_mat_q4(view, x, type=kind, ids=torch.from_numpy(e).cuda(), out=out[:, :N])
    check(out[:, :N], *want(w, x, kind, e.tolist()))
    assert bool((out[:, N:] == 3.0).all())


def test_same_rows_alone_and_together(gxlib, dev):
    """A row's result does not depend on the rows beside it (of the same number of columns at once)."""
    rng = np.random.default_rng(5)
    w = weights(rng, 4, 100, 512, Q4_0)
    x = torch.from_numpy(rng.standard_normal((8, 512))).cuda().to(F16)
    ids = torch.tensor([0, 1, 2, 3, 0, 1, 2, 3], dtype=torch.int32, device="cuda")
    both = gxlib.mul_mat_q4(w, x, type=Q4_0, ids=ids, out_dtype=F32)
    for j in range(8):
        assert torch.equal(gxlib.mul_mat_q4(w, x[j:j + 1], type=Q4_0, ids=ids[j:j + 1], out_dtype=F32), both[j:j + 1])
    assert torch.equal(gxlib.mul_mat_q4(w, x, type=Q4_0, ids=ids, out_dtype=F32), both)


@pytest.mark.parametrize("rows", [5, 40, 300])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_bad_rows_stay_alone(gxlib, dev, rows, bad):
    rng = np.random.default_rng(6)
    w = weights(rng, 1, 40, 256, Q4_1)
    x = torch.from_numpy(rng.standard_normal((rows, 256))).cuda().to(BF16)
    y, tol = want(w, x, Q4_1, [0] * rows)
    x[2, 100] = bad
    got = gxlib.mul_mat_q4(w, x, type=Q4_1, out_dtype=F32)
    assert not bool(torch.isfinite(got[2]).any())
    check(got, y, tol, torch.tensor([2], device="cuda"))


def test_reported(gxlib, dev):
    rng = np.random.default_rng(7)
    w = weights(rng, 4, 20, 64, Q4_0)
    x = torch.from_numpy(rng.standard_normal((6, 64))).cuda().to(F16)
    e = [0, 9, 3, -1, 4, 1]
    out = torch.full((6, 20), 5.0, dtype=F32, device="cuda")
    gxlib.mul_mat_q4(w, x, type=Q4_0, ids=torch.tensor(e, dtype=torch.int32, device="cuda"), out=out)
    assert error_code(gxlib) == 1 and error_code(gxlib) == 0
    y, tol = want(w, x, Q4_0, [v if v < 4 else -1 for v in e])
    left = torch.tensor([1, 3, 4], device="cuda")
    check(out, y, tol, left)
    assert bool((out[left] == 5.0).all())
    # borders that do not ascend: that group is left out, the others are there
    order = torch.arange(6, dtype=torch.int32, device="cuda")
    out.fill_(5.0)
    gxlib.mul_mat_q4(w, x, type=Q4_0, offsets=torch.tensor([0, 2, 1, 4, 6], dtype=torch.int32, device="cuda"), order=order, scatter=True, out=out)
    assert error_code(gxlib) == 1
    y, tol = want(w, x, Q4_0, [0, 2, 2, 2, 3, 3])
    check(out[[0, 2, 3, 4, 5]], y[[0, 2, 3, 4, 5]], tol[[0, 2, 3, 4, 5]])
    # borders outside the rows
    out.fill_(5.0)
    gxlib.mul_mat_q4(w, x, type=Q4_0, offsets=torch.tensor([-1, 2, 4, 6, 7], dtype=torch.int32, device="cuda"), order=order, scatter=True, out=out)
    assert error_code(gxlib) == 1
    y, tol = want(w, x, Q4_0, [-1, -1, 1, 1, 2, 2])
    check(out, y, tol, torch.tensor([0, 1], device="cuda"))
    assert bool((out[:2] == 5.0).all())
    # rows of x and of the result that do not exist
    out.fill_(5.0)
    gxlib.mul_mat_q4(w, x[:3], type=Q4_0, offsets=torch.tensor([0, 6, 6, 6, 6], dtype=torch.int32, device="cuda"),
                     order=torch.tensor([0, 1, 5, 2, -3, 77], dtype=torch.int32, device="cuda"), gather=1, scatter=True, n_rows=6, out=out)
    assert error_code(gxlib) == 1
    y, tol = want(w, x, Q4_0, [0] * 6)
    check(out[:3], y[:3], tol[:3])
    assert bool(torch.isnan(out[5]).all()) and bool((out[3:5] == 5.0).all())
    gxlib.mul_mat_q4(w, x, type=Q4_0, ids=torch.full((6,), -1, dtype=torch.int32, device="cuda"), out=out)
    assert error_code(gxlib) == 0


def test_graph_and_streams(gxlib, dev):
    """Captured and replayed on new ids and rows, and two streams at once."""
    rng = np.random.default_rng(8)
    E, N, K, T, k = 16, 96, 512, 4, 4
    gate, up, down = weights(rng, E, N, K, Q4_0), weights(rng, E, N, K, Q4_0), weights(rng, E, K, 64, Q4_0)
    x = torch.zeros((T, K), dtype=BF16, device="cuda")
    ids = torch.zeros((T, k), dtype=torch.int32, device="cuda")

    def layer():
        h = gxlib.mul_mat_q4_glu(gate, up, x, type=Q4_0, ids=ids, gather=k)
        return gxlib.mul_mat_q4(down, h[:, :64].contiguous(), type=Q4_0, ids=ids, out_dtype=F32)

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer()
    for _ in range(3):
        x.copy_(torch.from_numpy(rng.standard_normal((T, K))).cuda())
        ids.copy_(torch.from_numpy(rng.integers(0, E, (T, k)).astype(np.int32)).cuda())
        graph.replay()
        assert torch.equal(y, layer())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = [gxlib.mul_mat_q4(gate, x, type=Q4_0, ids=ids, gather=k) for _ in range(20)]
    b = [gxlib.mul_mat_q4(gate, x, type=Q4_0, ids=ids, gather=k, stream=side) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, a[0]) for t in a + b)


def test_far_weights(gxlib, dev):
    """Matrices that begin beyond 4 GiB."""
    rng = np.random.default_rng(9)
    E, N, K = 1300, 1536, 4096
    w = torch.zeros((E, N, K // 32 * 18), dtype=torch.uint8, device="cuda")
    last = weights(rng, 1, N, K, Q4_0)
    w[E - 1] = last[0]
    assert (E - 1) * N * w.shape[2] > 1 << 32
    x = torch.from_numpy(rng.standard_normal((40, K))).cuda().to(BF16)
    y, tol = want(last, x, Q4_0, [0] * 40)
    got = gxlib.mul_mat_q4(w, x[:2], type=Q4_0, ids=torch.tensor([E - 1, E - 1], dtype=torch.int32, device="cuda"), out_dtype=F32)
    check(got, y[:2], tol[:2])
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[E] = 40
    check(gxlib.mul_mat_q4(w, x, type=Q4_0, offsets=offsets, out_dtype=F32), y, tol)


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("K,N", [(256, 130), (320, 70), (1600, 40)])
def test_short_groups_among_long_ones(gxlib, dev, kind, dtype, out, K, N):
    """Groups of none, one, a few and hundreds of rows in one call: which kernel takes a group goes by its length, and tiles of few
    rows follow full ones (a CTA of a pair may then have no rows at all)."""
    rng = np.random.default_rng(K)
    sizes = [1, 0, 300, 2, 24, 25, 16, 17, 513, 3, 0, 8, 9, 70, 26, 1, 257, 33]
    E, P = len(sizes), sum(sizes)
    w = weights(rng, E, N, K, kind)
    offsets = torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)).cuda()
    order = torch.from_numpy(rng.permutation(P).astype(np.int32)).cuda()
    e = np.repeat(np.arange(E), sizes).tolist()
    x = torch.from_numpy(rng.standard_normal((P, K))).cuda().to(dtype)
    y, tol = want(w, x[order.long()], kind, e, out)
    for _ in range(3):
        check(gxlib.mul_mat_q4(w, x, type=kind, offsets=offsets, order=order, gather=1, out_dtype=out), y, tol)
        got = gxlib.mul_mat_q4(w, x[order.long()].contiguous(), type=kind, offsets=offsets, order=order, scatter=True, out_dtype=out)
        check(got[order.long()], y, tol)
    y, tol = want_glu(w, w.flip(0).contiguous(), x[order.long()], kind, e, 0, out)
    check(gxlib.mul_mat_q4_glu(w, w.flip(0).contiguous(), x, type=kind, offsets=offsets, order=order, gather=1, out_dtype=out), y, tol)
    assert error_code(gxlib) == 0


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("pad", [4, 16, 20])
def test_strides_of_many_rows(gxlib, dev, kind, pad):
    rng = np.random.default_rng(pad)
    G, N, K, T = 2, 77, 448, 150
    w = weights(rng, G, N, K, kind)
    rb = w.shape[2]
    wide = torch.zeros(G * (N * (rb + pad) + 4 * pad) + 64, dtype=torch.uint8, device="cuda")
    view = wide.as_strided((G, N, rb), (N * (rb + pad) + 4 * pad, rb + pad, 1))
    view.copy_(w)
    x = torch.from_numpy(rng.standard_normal((T, K + 24))).cuda().to(F16)[:, :K]
    out = torch.full((T, N + 5), 3.0, dtype=F16, device="cuda")
    offsets = torch.tensor([0, 60, 150], dtype=torch.int32, device="cuda")
    gxlib.mul_mat_q4(view, x, type=kind, offsets=offsets, out=out[:, :N])
    check(out[:, :N], *want(w, x, kind, [0] * 60 + [1] * 90, F16))
    assert bool((out[:, N:] == 3.0).all())


@pytest.mark.parametrize("K,rows,E", [(65536, 2, 1), (65536, 40, 1), (16384, 256, 3), (7168, 256, 2)])
def test_long_rows(gxlib, dev, K, rows, E):
    """The longest rows (of which shared memory holds one), and CTAs of fewer threads than ids."""
    rng = np.random.default_rng(K)
    w = weights(rng, E, 9, K, Q4_0)
    x = torch.from_numpy(rng.standard_normal((rows, K))).cuda().to(BF16)
    e = rng.integers(0, E, rows).astype(np.int32)
    if rows <= 256:
        check(gxlib.mul_mat_q4(w, x, type=Q4_0, ids=torch.from_numpy(e).cuda(), out_dtype=F32), *want(w, x, Q4_0, e.tolist()))
    if E == 1:
        check(gxlib.mul_mat_q4(w, x, type=Q4_0, out_dtype=F32), *want(w, x, Q4_0, e.tolist()))
    assert error_code(gxlib) == 0


def test_many_rows_captured_and_beside_another_stream(gxlib, dev):
    rng = np.random.default_rng(12)
    E, N, K, T, k = 8, 200, 512, 120, 4
    w = weights(rng, E, N, K, Q4_0)
    x = torch.zeros((T, K), dtype=BF16, device="cuda")
    ids = torch.zeros((T, k), dtype=torch.int32, device="cuda")

    def step(stream=None):
        order, offsets = gxlib.group_rows(ids, E, stream=stream)
        return gxlib.mul_mat_q4(w, x, type=Q4_0, offsets=offsets, order=order, gather=k, scatter=True, stream=stream)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for _ in range(3):
        x.copy_(torch.from_numpy(rng.standard_normal((T, K))).cuda())
        ids.copy_(torch.from_numpy(rng.integers(0, E, (T, k)).astype(np.int32)).cuda())
        graph.replay()
        assert torch.equal(y, step())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = [step(s) for _ in range(10) for s in (None, side)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, y) for t in got)


def test_products_on_the_slots_of_an_arena(gxlib, dev, tmp_path):
    """A checkpoint of Q4_0 and Q4_1 experts, its records in an arena, the slots the products' matrices."""
    import ctypes as C
    from gguf import GGMLQuantizationType, GGUFWriter
    from galactus_b200.models import ModelShape
    H, I, E = 128, 192, 5
    rng = np.random.default_rng(13)
    f = GGUFWriter(str(tmp_path / "m.gguf"), "qwen3moe")
    f.add_block_count(1)
    f.add_expert_count(E)
    f.add_expert_used_count(2)
    held = {}
    for role, n, m, kind in (("down", H, I, Q4_1), ("gate", I, H, Q4_0), ("up", I, H, Q4_0)):
        held[role] = weights(rng, E, n, m, kind)
        f.add_tensor(f"blk.0.ffn_{role}_exps.weight", held[role].cpu().numpy(), raw_dtype=GGMLQuantizationType(kind))
    f.write_header_to_file()
    f.write_kv_data_to_file()
    f.write_tensors_to_file()
    f.close()
    m = ModelShape("q4", 1, H, E, 2, I, Q4_0, Q4_0, Q4_1)
    arena = gxlib.Arena(m, capacity_bytes=E * m.record, policy=gxlib.POLICY_AUTO, max_tokens=8)
    try:
        n = C.c_uint32()
        gxlib.check(gxlib.lib().gx_arena_load_gguf(arena.h, str(tmp_path / "m.gguf").encode(), C.byref(n)), "gx_arena_load_gguf")
        assert n.value == E
        stream = torch.cuda.current_stream()
        arena.warm_all(stream)
        base, record, slots = arena.layer_view(0)
        e = [3, 0, 4, 3, 1]
        ids = torch.tensor([arena.slot_of(0, v) for v in e], dtype=torch.int32, device="cuda")
        x = torch.from_numpy(rng.standard_normal((5, H))).cuda().to(BF16)
        h = torch.empty((5, I), dtype=F16, device="cuda")
        lib, s = gxlib.lib(), stream.cuda_stream
        gxlib.check(lib.gx_mul_mat_q4_glu(Q4_0, base + m.off_gate, base + m.off_up, H, I, H // 32 * 18, record, slots, 30, x.data_ptr(), 5,
                                          2 * H, ids.data_ptr(), None, None, 5, 1, 0, 0, 0.0, 0.0, 1, h.data_ptr(), 2 * I, s))
        check(h, *want_glu(held["gate"], held["up"], x, Q4_0, e, 0, F16))
        y = torch.empty((5, H), device="cuda")
        gxlib.check(lib.gx_mul_mat_q4(Q4_1, base, I, H, I // 32 * 20, record, slots, 1, h.data_ptr(), 5, 2 * I, ids.data_ptr(), None, None, 5, 1,
                                      0, 0, y.data_ptr(), 4 * H, s))
        check(y, *want(held["down"], h, Q4_1, e))
    finally:
        arena.close()


def test_python_refusals(gxlib, dev):
    rng = np.random.default_rng(10)
    w = weights(rng, 2, 8, 64, Q4_0)
    x = torch.zeros((3, 64), dtype=BF16, device="cuda")
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (lambda: gxlib.mul_mat_q4(w, x, type=Q4_1, ids=ids), lambda: gxlib.mul_mat_q4(w, x, type=8, ids=ids),
                lambda: gxlib.mul_mat_q4(w.int(), x, type=Q4_0, ids=ids), lambda: gxlib.mul_mat_q4(w, x, type=Q4_0, ids=ids.long()),
                lambda: gxlib.mul_mat_q4(w, x, type=Q4_0, ids=ids, offsets=ids), lambda: gxlib.mul_mat_q4(w, x, type=Q4_0, ids=ids, n_rows=4),
                lambda: gxlib.mul_mat_q4(w, x, type=Q4_0, ids=ids, out_dtype=torch.int32),
                lambda: gxlib.mul_mat_q4(w, x.cpu(), type=Q4_0, ids=ids), lambda: gxlib.mul_mat_q4_glu(w, w[:1], x, type=Q4_0, ids=ids)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(gxlib.GxError):
        gxlib.mul_mat_q4(w, x, type=Q4_0)                       # two matrices, none named
    with pytest.raises(gxlib.GxError):
        gxlib.mul_mat_q4(w, x.float(), type=Q4_0, ids=ids, out_dtype=F32)
    assert gxlib.mul_mat_q4(w, x[:0], type=Q4_0, ids=ids[:0]).shape == (0, 8)


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,K", [(3, 7168), (40, 1024), (40, 4096)])
def test_sums_of_one_sign(gxlib, dev, kind, dtype, rows, K):
    """Positive rows (and, with Q4_1, positive weights): what the sums cut off does not cancel."""
    rng = np.random.default_rng(K + rows)
    w = weights(rng, 1, 40, K, kind)
    if kind == Q4_1:
        b = w.view(1, 40, K // 32, BLOCK[kind])
        b[..., 1] &= 127                                       # (the signs of d and m)
        b[..., 3] &= 127
    x = torch.from_numpy(0.5 + np.abs(rng.standard_normal((rows, K)))).cuda().to(dtype)
    got = gxlib.mul_mat_q4(w, x, type=kind, out_dtype=F32)
    check(got, *want(w, x, kind, [0] * rows), rms=None)


@pytest.mark.parametrize("T,k", [(3, 4), (20, 3)])
@pytest.mark.parametrize("scatter", [False, True])
def test_one_matrix_in_an_order(gxlib, dev, T, k, scatter):
    """Neither ids nor offsets, but an order: rows of x by order[j] // gather, results in place or scattered."""
    rng = np.random.default_rng(T)
    K, N = 256, 70
    w = weights(rng, 1, N, K, Q4_0)
    x = torch.from_numpy(rng.standard_normal((T, K))).cuda().to(BF16)
    order = rng.permutation(T * k).astype(np.int32)
    got = gxlib.mul_mat_q4(w, x, type=Q4_0, order=torch.from_numpy(order).cuda(), gather=k, scatter=scatter, out_dtype=F32)
    if scatter:
        got = got[torch.from_numpy(order).long().cuda()]
    check(got, *want(w, x[torch.from_numpy(order // k).long().cuda()], Q4_0, [0] * (T * k)))
    assert error_code(gxlib) == 0
