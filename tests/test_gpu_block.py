"""The norms around a block on the GPU against the formula in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
EPS = 1e-6
U = 2.0 ** -24


def rand(rng, *shape, dtype=F32, scale=1.0):
    return torch.from_numpy(scale * rng.standard_normal(shape)).cuda().to(dtype)


def unit(x, weight, eps=EPS):
    x = x.double()
    return x / torch.sqrt(x.square().mean(1, keepdim=True) + eps) * (1.0 if weight is None else weight.double())


def close(got, want, tol):
    """Within tol, and half a step of the result's type."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bad = ~((got.double() - want).abs() <= tol * (1 + half) + half * want.abs() + tiny)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, at {bad.nonzero()[:4].tolist()}"


WIDTHS = [1, 7, 8, 64, 100, 1024, 2048, 2880, 4095, 7168, 16384, 65536]


@pytest.mark.parametrize("dtype,out", [(F32, BF16), (F32, F32), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("H", WIDTHS)
def test_rms_norm(gxlib, dev, dtype, out, H):
    """The root of a sum of H rounded squares is off by (H / 512 + 20) half steps at most (each thread adds 16 at most in a
    chain, then 5 + 16 + 8 values), the quotient, the root and two products by half a step each."""
    rng = np.random.default_rng(H)
    for T in (1, 2, 5, 160, 400 if H < 9000 else 3):
        x = rand(rng, T, H, dtype=dtype, scale=3.0)
        w = rand(rng, H)
        want = unit(x, w)
        close(gxlib.rms_norm(x, w, eps=EPS, out_dtype=out), want, want.abs() * 64 * U)
        want = unit(x, None, 1e-2)
        close(gxlib.rms_norm(x, eps=1e-2, out_dtype=out), want, want.abs() * 64 * U)


def test_rms_norm_many_rows(gxlib, dev):
    rng = np.random.default_rng(1)
    x = rand(rng, 3000, 333, dtype=BF16)
    want = unit(x, None)
    close(gxlib.rms_norm(x, eps=EPS), want, want.abs() * 64 * U)
    # rows further apart, results in place and between guards
    wide = rand(rng, 40, 136)
    x = wide[:, :128]
    keep, want = wide.clone(), unit(x, None)
    out = torch.full((40, 200), 3.0, device="cuda")
    gxlib.rms_norm(x, eps=EPS, out=out[:, 8:136])
    close(out[:, 8:136], want, want.abs() * 64 * U)
    assert bool((out[:, :8] == 3.0).all()) and bool((out[:, 136:] == 3.0).all())
    gxlib.rms_norm(x, eps=EPS, out=x)
    assert torch.equal(x, out[:, 8:136]) and torch.equal(wide[:, 128:], keep[:, 128:])
    # rows on odd addresses of their type
    x = wide.reshape(-1)[1:1 + 40 * 128].view(40, 128)
    want = unit(x, None)
    close(gxlib.rms_norm(x, eps=EPS), want, want.abs() * 64 * U)


def test_zero_rows(gxlib, dev):
    x = torch.zeros((3, 64), device="cuda")
    assert bool((gxlib.rms_norm(x) == 0).all())
    assert gxlib.rms_norm(x[:0]).shape == (0, 64)


def formula(y, weights, ids, shared, shared_gate, norm, gate, sigmoid, scale, residual):
    """(out, how far f32 may be off): every rounding is half a step of a partial sum of magnitudes."""
    T, k, H = y.shape
    m = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(m)
    for s in range(k):
        row = y[:, s].double()
        if weights is not None:
            row = row * weights[:, s, None].double()
        if ids is not None:
            row = torch.where(ids[:, s, None] >= 0, row, 0.0)
        m, mag = m + row, mag + row.abs()
    if shared is not None:
        row = shared.double()
        if shared_gate is not None:
            row = row * torch.sigmoid(shared_gate.double())[:, None]
        m, mag = m + row, mag + row.abs()
    err = mag * (2 * k + 8) * U                                   # (a sigmoid is within 4 steps)
    if norm is not None:
        root = torch.sqrt(m.square().mean(1, keepdim=True) + EPS)
        err = err / root + m.abs() / root * (err.square().mean(1, keepdim=True).sqrt() / root + 64 * U)
        err = err * norm.double().abs()
        m = m / root * norm.double()
    if gate is not None:
        g = torch.sigmoid(gate.double()) if sigmoid else gate.double()
        m, err = m * g, (err + m.abs() * 9 * U) * g.abs()
    r = residual.double() if residual is not None else 0.0
    out = r + scale * m
    return out, abs(scale) * (err + m.abs() * 2 * U) + out.abs() * U


CASES = [dict(), dict(routed=True), dict(routed=True, drop=True, shared=True), dict(routed=True, shared=True, gated=True, post=True),
         dict(routed=True, drop=True, shared=True, gated=True, post=True, gate="channel", scale=0.22, residual=True, next=True),
         dict(post=True, gate="row", sigmoid=True, residual=True, next=True), dict(gate="full", scale=-2.0, residual=True),
         dict(gate="one", sigmoid=True, next=True), dict(routed=True, residual=True, next=True)]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("kind,res,out,nxt", [(F32, F32, F32, BF16), (BF16, F32, F32, F16), (F16, F16, F16, F16), (F32, BF16, BF16, F32)])
@pytest.mark.parametrize("T,k,H", [(1, 8, 2048), (1, 1, 1), (3, 2, 65), (5, 8, 2880), (200, 4, 520), (2, 3, 20000), (700, 3, 512),
                                   (431, 2, 1032), (300, 33, 520), (310, 4, 8192)])
def test_block_out(gxlib, dev, case, kind, res, out, nxt, T, k, H):
    c = CASES[case]
    rng = np.random.default_rng(case * 100 + T + H)
    y = rand(rng, T, k, H, dtype=kind)
    weights = torch.softmax(rand(rng, T, k), 1).contiguous() if c.get("routed") else None
    ids = None
    if c.get("drop"):
        ids = torch.from_numpy(rng.integers(-1, 3, (T, k)).astype(np.int32)).cuda()
        ids[T // 2] = -1                                          # a row that nothing is left of
        y[ids < 0] = float("nan")
    shared = rand(rng, T, H, dtype=kind) if c.get("shared") else None
    shared_gate = rand(rng, T) if c.get("gated") else None
    norm = rand(rng, H) if c.get("post") else None
    gate = {None: None, "row": (T, 1), "channel": (1, H), "full": (T, H), "one": (1, 1)}[c.get("gate")]
    gate = rand(rng, *gate) if gate else None
    residual = rand(rng, T, H, dtype=res, scale=3.0) if c.get("residual") else None
    weight = rand(rng, H) if c.get("next") else None
    got = gxlib.block_out(y, weights=weights, ids=ids, shared=shared, shared_gate=shared_gate, norm=norm, eps=EPS, gate=gate,
                          gate_sigmoid=c.get("sigmoid", False), scale=c.get("scale", 1.0), residual=residual, out_dtype=out,
                          next_norm=weight, next_dtype=nxt if c.get("next") else None)
    want, err = formula(y, weights, ids, shared, shared_gate, norm, gate, c.get("sigmoid", False), c.get("scale", 1.0), residual)
    if c.get("next"):
        got, after = got
        assert after.dtype == nxt
        root = torch.sqrt(want.square().mean(1, keepdim=True) + EPS)
        normed = unit(want, weight)
        rel = err.square().mean(1, keepdim=True).sqrt() / root + 64 * U
        close(after, normed, err / root * weight.double().abs() + normed.abs() * rel)
    assert got.dtype == out
    close(got, want, err)


@pytest.mark.parametrize("case", [1, 4, 5, 8])
@pytest.mark.parametrize("kind,res,out,nxt", [(F32, F32, F32, BF16), (BF16, F32, F32, F16), (F16, F16, F16, F16)])
@pytest.mark.parametrize("T,k,H", [(3, 2, 8), (77, 3, 256), (9, 40, 136), (2048, 2, 512), (2047, 2, 512), (2100, 35, 264), (5000, 1, 64),
                                   (300, 3, 4096), (512, 8, 2048), (511, 8, 2048), (300, 33, 4096), (20, 2, 4104), (74, 2, 4104), (75, 2, 4104)])
def test_block_out_beside_the_borders(gxlib, dev, case, kind, res, out, nxt, T, k, H):
    """On both sides of what chooses a warp, a CTA, a cluster per row, or rings of rows."""
    test_block_out(gxlib, dev, case, kind, res, out, nxt, T, k, H)


def test_equals_combine(gxlib, dev):
    """The weighted sum alone has gx_combine's bits."""
    rng = np.random.default_rng(3)
    T, k, H = 9, 8, 2048
    y, w = rand(rng, T, k, H), torch.softmax(rand(rng, T, k), 1).contiguous()
    want = torch.empty((T, H), device="cuda")
    gxlib.check(gxlib.lib().gx_combine(y.data_ptr(), w.data_ptr(), want.data_ptr(), H, k, T, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(gxlib.block_out(y, weights=w), want)


def test_in_place_and_strides(gxlib, dev):
    rng = np.random.default_rng(4)
    T, k, H = 33, 4, 512
    wide = rand(rng, T, k + 1, H + 8, dtype=BF16)
    y, w, res = wide[:, :k, :H], torch.softmax(rand(rng, T, k), 1).contiguous(), rand(rng, T, H)
    want, err = formula(y, w, None, None, None, None, None, False, 0.5, res)
    out, after = gxlib.block_out(y, weights=w, scale=0.5, residual=res, next_dtype=BF16)
    close(out, want, err)
    assert torch.equal(after, gxlib.block_out(y, weights=w, scale=0.5, residual=res, out=res, next_dtype=BF16)[1]) and torch.equal(out, res)
    assert torch.equal(gxlib.rms_norm(out, out_dtype=BF16), after)
    assert gxlib.block_out(y[:0], weights=w[:0]).shape == (0, H)


def test_graph(gxlib, dev):
    rng = np.random.default_rng(5)
    y, w, res = rand(rng, 1, 8, 2048), torch.softmax(rand(rng, 1, 8), 1).contiguous(), rand(rng, 1, 2048)

    def step():
        h = gxlib.rms_norm(res, out_dtype=BF16)
        return (h,) + gxlib.block_out(y, weights=w, residual=res, next_dtype=BF16)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        for t in (y, res):
            t.copy_(rand(rng, *t.shape))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_python_refusals(gxlib, dev):
    y, w = torch.zeros((3, 2, 64), device="cuda"), torch.zeros((3, 2), device="cuda")
    for bad in (dict(weights=w[:2]), dict(weights=w.double()), dict(ids=w), dict(shared=y[:, 0, :32]), dict(residual=y), dict(norm=w),
                dict(gate=w), dict(gate=w.half()), dict(out=y), dict(out_dtype=torch.int32), dict(next_norm=w), dict(shared=y[:, 0], shared_gate=w)):
        with pytest.raises(ValueError):
            gxlib.block_out(y, **bad)
    with pytest.raises(gxlib.GxError):
        gxlib.block_out(y.double(), out_dtype=F32)
    with pytest.raises(gxlib.GxError):
        gxlib.rms_norm(w, eps=-1.0)


@pytest.mark.parametrize("T", [1, 5, 300])
def test_layer(gxlib, dev, T):
    """A block as it is used: norm, router, gated products, down products, weighted sum with the shared expert, residual, next norm."""
    from test_gpu_q4 import Q4_0, parts, weights
    rng = np.random.default_rng(T)
    H, I, E, k = 512, 256, 16, 4
    x, w0, w1 = rand(rng, T, H, scale=2.0), 1.0 + 0.1 * rand(rng, H), 1.0 + 0.1 * rand(rng, H)
    gate, up, down = weights(rng, E, I, H, Q4_0), weights(rng, E, I, H, Q4_0), weights(rng, E, H, I, Q4_0)
    sg, su, sd = weights(rng, 1, I, H, Q4_0), weights(rng, 1, I, H, Q4_0), weights(rng, 1, H, I, Q4_0)
    wr, ws = rand(rng, E, H, scale=0.05), rand(rng, H, scale=0.05)

    h = gxlib.rms_norm(x, w0, eps=EPS, out_dtype=BF16)
    logits = h.float() @ wr.T
    ids = torch.empty((T, k), dtype=torch.int32, device="cuda")
    probs = torch.empty((T, k), device="cuda")
    import ctypes as C
    desc = gxlib._lib.gx_router_desc(0, E, k, 1, 1, 1, 0, 1.0)
    gxlib.check(gxlib.lib().gx_router_forward(C.byref(desc), logits.data_ptr(), E, 0, T, 1, ids.data_ptr(), probs.data_ptr(), 0, 0,
                                              torch.cuda.current_stream().cuda_stream))
    if T * k <= 256:
        a = gxlib.mul_mat_q4_glu(gate, up, h, type=Q4_0, ids=ids, gather=k)
        y = gxlib.mul_mat_q4(down, a, type=Q4_0, ids=ids, out_dtype=F32)
    else:
        order, offsets = gxlib.group_rows(ids, E)
        a = gxlib.mul_mat_q4_glu(gate, up, h, type=Q4_0, offsets=offsets, order=order, gather=k)
        y = gxlib.mul_mat_q4(down, a, type=Q4_0, offsets=offsets, order=order, scatter=True, out_dtype=F32)
    s = gxlib.mul_mat_q4(sd, gxlib.mul_mat_q4_glu(sg, su, h, type=Q4_0), type=Q4_0, out_dtype=F32)
    out, after = gxlib.block_out(y.view(T, k, H), weights=probs, ids=ids, shared=s, shared_gate=h.float() @ ws, residual=x,
                                 next_norm=w1, next_dtype=BF16)

    # The formula on the same routes, with a rounding to BF16 where the layer has one. An activation that f32 sums put at the other
    # side of a border is off by two roundings, each half a step, 2^-8 of the value at most: taken as independent errors, of a
    # variance of (2^-8)^2 / 3 of its square each. Of 150 thousand results none is six deviations off.
    h64 = unit(x, w0).to(BF16).double()
    e64 = torch.topk(h64 @ wr.double().T, k, dim=1).indices
    assert torch.equal(e64.sort(1).values, ids.long().sort(1).values)
    p64 = torch.softmax(h64 @ wr.double().T, 1).gather(1, ids.long())
    p64 = p64 / p64.sum(1, keepdim=True)
    step = (2.0 ** -8) ** 2 / 3

    def ffn(rows, gm, um, dm):
        gm, um, dm = (parts(m, Q4_0)[0] for m in (gm, um, dm))
        g, u = rows @ gm.T, rows @ um.T
        act = g * torch.sigmoid(g) * u
        return act.to(BF16).double() @ dm.T, (2 * step * act ** 2) @ (dm ** 2).T

    want, var = x.double().clone(), torch.zeros((T, H), dtype=torch.float64, device="cuda")
    for e in range(E):
        t, sl = (ids == e).nonzero(as_tuple=True)
        if len(t):
            y64, v64 = ffn(h64[t], gate[e], up[e], down[e])
            want.index_add_(0, t, p64[t, sl][:, None] * y64)
            var.index_add_(0, t, p64[t, sl][:, None] ** 2 * v64)
    y64, v64 = ffn(h64, sg[0], su[0], sd[0])
    weight = torch.sigmoid(h64 @ ws.double())[:, None]
    want, var = want + weight * y64, var + weight ** 2 * v64
    assert bool(((out.double() - want).abs() <= 6 * var.sqrt() + want.abs() * 2.0 ** -20).all())
    close(after, unit(out, w1), unit(out, w1).abs() * 64 * U)
