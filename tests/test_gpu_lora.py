"""Low-rank deltas of many adapters (gx_lora_mul_mat) against the float64
definition, at the sizes, ranks and masks where they can go wrong."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def acc_bound(K: int) -> float:
    """Of an f32 sum of K exact products, relative to the sum of their magnitudes: one rounding or truncation (2^-23) of
    the sum per 16 products, and the alignment of the 16 (as much each)."""
    return (K / 16 + 16) * 2.0 ** -23


def make(T, k, n_as, adapters, rank, K, N, kind, out, seed, amp=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
    G = n_as * adapters
    b = (rnd(G, N, (rank + 7) // 8 * 8) * 0.1).to(TYPES[kind])[:, :, :rank]             # rows of 16-byte multiples
    return dict(a=(rnd(G, rank, K) * K ** -0.5).to(TYPES[kind]), b=b,
                x=(rnd(T, K) * amp).to(TYPES[kind]), base=rnd(T * k, N).to(TYPES[out]))


def reference(s, keys, k, n_as, ranks, scale):
    """float64 result and error bound before the final rounding, row by row of base."""
    want, tol = s["base"].double().clone(), torch.zeros_like(s["base"], dtype=torch.float64)
    for g in np.unique(keys[keys >= 0]).tolist():
        rows = torch.from_numpy(np.nonzero(keys == g)[0]).cuda()
        r, sc = int(ranks[g // n_as]), float(scale[g // n_as])
        if r == 0:
            continue
        x, a, b = s["x"][rows // k].double(), s["a"][g, :r].double(), s["b"][g, :, :r].double()
        h = sc * (x @ a.T)
        # f32 sums of up to eight parts of K, the scale; split into parts of 22 bits
        eh = abs(sc) * (x.abs() @ a.abs().T) * (acc_bound(x.shape[1]) + 10 * 2.0 ** -24) + 2.0 ** -22 * h.abs()
        want[rows] += h @ b.T
        tol[rows] = eh @ b.abs().T + (h.abs() @ b.abs().T) * acc_bound(48 * ((r + 15) // 16))
    return want, tol


def compare(got, want, tol, kind):
    err = (got.double() - want).abs()
    lim = tol + (2.0 ** -24 + HALF[kind]) * (want.abs() + tol) + (2.0 ** -25 if kind == "f16" else 0.0)
    bad = ~(err <= lim)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / lim).max()):.3g} of the bound"


def keys_of(ids, adapter, n_as):
    a = adapter.astype(np.int64)[:, None]
    return np.where((a < 0) | (ids < 0), -1, a * n_as + ids).reshape(-1)


CASES = [
    # T, k, experts, adapters, rank, mixed, K, N, type, out
    (1, 1, 1, 1, 16, False, 2048, 2048, "f16", "f32"),
    (1, 1, 1, 3, 8, False, 64, 128, "bf16", "bf16"),
    (2, 1, 1, 2, 1, False, 8, 1, "f16", "f16"),
    (64, 1, 1, 48, 64, True, 1024, 1000, "bf16", "bf16"),
    (65, 1, 1, 2, 16, False, 72, 129, "f16", "f32"),
    (130, 1, 1, 1, 128, True, 520, 384, "bf16", "f32"),
    (37, 4, 6, 5, 24, True, 200, 257, "f16", "f32"),
    (300, 8, 32, 4, 16, False, 256, 192, "bf16", "f32"),
    (1000, 1, 1, 3, 32, True, 4096, 640, "f16", "f16"),
    (9, 2, 3, 700, 72, True, 136, 65, "bf16", "f32"),
    (3000, 1, 1, 40, 40, True, 192, 300, "f16", "f32"),
    (2500, 4, 30, 5, 64, True, 512, 136, "bf16", "bf16"),
]


@pytest.mark.parametrize("T,k,n_as,adapters,rank,mixed,K,N,kind,out", CASES)
def test_deltas(gxlib, dev, T, k, n_as, adapters, rank, mixed, K, N, kind, out):
    from galactus_b200.moe import device_error
    device_error()
    rng = np.random.default_rng(T + K)
    s = make(T, k, n_as, adapters, rank, K, N, kind, out, T + N)
    ids = rng.integers(0, n_as, size=(T, k)).astype(np.int32)
    adapter = rng.integers(-1 if T > 2 else 0, adapters, size=T).astype(np.int32)
    ranks = rng.integers(0 if T > 2 else 1, rank + 1, size=adapters).astype(np.int32) if mixed else np.full(adapters, rank, np.int32)
    scale = rng.uniform(0.25, 3.0, size=adapters).astype(np.float32)
    if mixed:
        # what lies behind an adapter's rank is not read as numbers
        for g in range(n_as * adapters):
            s["a"][g, ranks[g // n_as]:] = float("nan")
            s["b"][g, :, ranks[g // n_as]:] = float("nan")
    dev_ids = torch.from_numpy(ids).cuda() if n_as > 1 or k > 1 else None
    order, offsets = gxlib.group_rows(dev_ids, n_as, adapter=torch.from_numpy(adapter).cuda(), n_adapters=adapters)
    kw = dict(order=order, gather=k, n_as=n_as, ranks=torch.from_numpy(ranks).cuda() if mixed else None,
              scale=torch.from_numpy(scale).cuda())
    want, tol = reference(s, keys_of(ids, adapter, n_as), k, n_as, ranks, scale)
    got = gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, base=s["base"], **kw)
    compare(got, want, tol, out)
    assert torch.equal(got, gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, base=s["base"], **kw))    # the same bits again
    # in place, inside wider rows, nothing else touched
    wide = torch.full((T * k + 2, N + 5), 9.0, dtype=TYPES[out], device="cuda")
    view = wide[1:-1, 2:N + 2]
    view.copy_(s["base"])
    gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, base=view, out=view, **kw)
    assert torch.equal(view, got)
    view.fill_(9.0)
    assert bool((wide == 9.0).all())
    assert device_error() == 0


def test_rows_in_place_without_scale(gxlib, dev):
    """No order: the rows already lie by adapter; rows behind the last group are copied."""
    s = make(50, 1, 1, 3, 16, 320, 256, "bf16", "f32", 3)
    offsets = torch.tensor([0, 7, 7, 41], dtype=torch.int32, device="cuda")
    keys = np.array([0] * 7 + [2] * 34 + [-1] * 9)
    want, tol = reference(s, keys, 1, 1, [16] * 3, [1.0] * 3)
    compare(gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, base=s["base"]), want, tol, "f32")


def test_large_h_in_f16(gxlib, dev):
    """h beyond the largest F16 number, and rows of very different size in one tile."""
    s = make(40, 1, 1, 1, 16, 512, 200, "f16", "f32", 8)
    s["x"] *= torch.logspace(-3, 4, 40, device="cuda")[:, None].half()
    offsets = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    scale = torch.tensor([64.0], device="cuda")
    keys = np.zeros(40, np.int64)
    assert float((64.0 * s["x"].float() @ s["a"][0].float().T).abs().max()) > 65504
    want, tol = reference(s, keys, 1, 1, [16], [64.0])
    compare(gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, base=s["base"], scale=scale), want, tol, "f32")


def test_nan_stays_in_its_row_and_adapter(gxlib, dev):
    s = make(20, 1, 1, 2, 16, 128, 160, "bf16", "f32", 4)
    offsets = torch.tensor([0, 11, 20], dtype=torch.int32, device="cuda")
    keys = np.array([0] * 11 + [1] * 9)
    want, tol = reference(s, keys, 1, 1, [16, 16], [1.0, 1.0])
    s["x"][3, 5] = float("nan")
    s["a"][1, 4, 7] = float("inf")
    got = gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, base=s["base"])
    rows = [i for i in range(11) if i != 3]
    compare(got[rows], want[rows], tol[rows], "f32")
    assert bool(torch.isnan(got[3]).all()) and not bool(torch.isfinite(got[11:]).any())


def test_errors_found_on_the_device(gxlib, dev):
    from galactus_b200.moe import device_error
    device_error()
    s = make(10, 1, 1, 2, 8, 64, 64, "f16", "f32", 6)
    cuda = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    good = gxlib.lora_mul_mat(s["a"], s["b"], s["x"], cuda([0, 4, 10]), base=s["base"])
    assert device_error() == 0
    got = gxlib.lora_mul_mat(s["a"], s["b"], s["x"], cuda([0, 4, 10]), base=s["base"], ranks=cuda([8, 9]))
    assert device_error() == 1 and torch.equal(got[:4], good[:4]) and torch.equal(got[4:], s["base"][4:])
    out = torch.full_like(s["base"], 5.0)
    gxlib.lora_mul_mat(s["a"], s["b"], s["x"], cuda([0, 4, 3]), base=s["base"], out=out)
    assert device_error() == 1 and torch.equal(out[:3], good[:3])
    out.fill_(5.0)
    order = cuda([0, 1, 2, 3, 4, 10, -1, 7, 8, 9])
    gxlib.lora_mul_mat(s["a"], s["b"], s["x"], cuda([0, 4, 10]), order=order, base=s["base"], out=out)
    assert device_error() == 1 and bool((out[5:7] == 5.0).all())
    keep = [i for i in range(10) if i not in (5, 6)]
    assert torch.equal(out[keep], good[keep])
    got = gxlib.lora_mul_mat(s["a"], s["b"], s["x"][:7], cuda([0, 4, 10]), base=s["base"])
    assert device_error() == 1 and torch.equal(got[:7], good[:7]) and bool(torch.isnan(got[7:]).all())


def test_adapters_beside_quantised_experts(gxlib, dev, orc):
    """As it is used: gx_mul_mat_id on Q8_0 experts, then the requests' adapters
    on its f32 output in place, and again in a captured graph."""
    from galactus_b200 import moe
    T, k, E, K, N, adapters, rank = 12, 2, 5, 256, 128, 3, 16
    rec = torch.empty((E, N, gxlib.row_bytes(gxlib.TYPE_Q8_0, K)), dtype=torch.uint8, device="cuda")
    gxlib.check(gxlib.lib().gx_synth_weights(gxlib.TYPE_Q8_0, rec.data_ptr(), K, E * N, 3, 0, 0.05, None))
    s = make(T, k, E, adapters, rank, K, N, "bf16", "f32", 5)
    x = s["x"].float()
    rng = np.random.default_rng(2)
    ids = rng.integers(0, E, size=(T, k)).astype(np.int32)
    adapter = rng.integers(-1, adapters, size=T).astype(np.int32)
    dids, dad = torch.from_numpy(ids).cuda(), torch.from_numpy(adapter).cuda()
    y = torch.empty((T * k, N), device="cuda")
    stream = torch.cuda.current_stream()

    def step(stream):
        rb = gxlib.row_bytes(gxlib.TYPE_Q8_0, K)
        moe.mul_mat_id(gxlib.TYPE_Q8_0, rec, K, N, rb, rb * N, E, x, 1, T, 4 * K, 4 * K, dids, k, T, 4 * k, y, stream=stream)
        base = y.clone()
        order, offsets = gxlib.group_rows(dids, E, adapter=dad, n_adapters=adapters)
        gxlib.lora_mul_mat(s["a"], s["b"], gxlib.round_rows(x, torch.bfloat16), offsets, order=order, gather=k, n_as=E,
                           base=y, out=y)
        return base
    s["base"] = step(stream)
    want, tol = reference(s, keys_of(ids, adapter, E), k, E, [rank] * adapters, [1.0] * adapters)
    compare(y, want, tol, "f32")
    first = y.clone()
    side = torch.cuda.Stream()
    side.wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(side)
    y.zero_()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first)


def test_wrapper_checks(gxlib, dev):
    s = make(10, 1, 1, 2, 8, 64, 64, "f16", "f32", 6)
    off = torch.tensor([0, 4, 10], dtype=torch.int32, device="cuda")
    ok = dict(base=s["base"])
    for bad in (dict(a=s["a"].bfloat16()), dict(x=s["x"][:, :32]), dict(b=s["b"][:, :32]), dict(b=s["b"].transpose(1, 2)),
                dict(offsets=off[:-1]), dict(order=off), dict(ranks=off), dict(scale=off[:2]), dict(out=s["base"].half()),
                dict(base=s["base"][:, :60]), dict(x=s["x"].cpu()), dict(n_as=3)):
        kw = {**dict(a=s["a"], b=s["b"], x=s["x"], offsets=off, **ok), **bad}
        with pytest.raises(ValueError):
            gxlib.lora_mul_mat(kw.pop("a"), kw.pop("b"), kw.pop("x"), kw.pop("offsets"), **kw)
