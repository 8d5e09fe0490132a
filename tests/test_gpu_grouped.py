"""Row grouping and the grouped products with unquantised experts against plain
float64 definitions, at the sizes where they can go wrong."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}      # half a step, relative


def acc_bound(K: int) -> float:
    """Of the f32 sum of K products, relative to the sum S of their magnitudes:
    the products are exact in f32; a step adds 16 of them to the running sum,
    each aligned to the largest (off by at most one f32 step of it, 16 times
    2^-23), and rounds or truncates the sum (2^-23 S) once per step."""
    return (K / 16 + 16) * 2.0 ** -23


# ------------------------------------------------------------------ grouping
def group_ref(ids, n_as, adapter, n_adapters):
    T, k = ids.shape
    key = ids.astype(np.int64)
    G = n_as * max(1, n_adapters)
    if adapter is not None:
        a = adapter.astype(np.int64)[:, None]
        key = np.where((a < 0) | (key < 0), -1, a * n_as + key)
    key = key.reshape(-1)
    order = np.argsort(np.where(key < 0, G, key), kind="stable")
    return order.astype(np.int32), np.concatenate([[0], np.cumsum(np.bincount(key[key >= 0], minlength=G))]).astype(np.int32)


@pytest.mark.parametrize("T,k,n_as,n_adapters", [
    (1, 1, 1, 0), (1, 8, 128, 0), (3, 4, 5, 0), (31, 1, 7, 3), (33, 8, 64, 0), (256, 8, 128, 0), (257, 8, 128, 0),
    (517, 8, 64, 24), (2048, 8, 128, 0), (5000, 3, 1, 11), (16384, 8, 256, 0), (700, 2, 8192, 0), (4099, 1, 1, 8192),
    (100, 8, 1024, 8),
])
def test_group_rows(gxlib, dev, T, k, n_as, n_adapters):
    rng = np.random.default_rng(T * 31 + k)
    ids = rng.integers(-1 if T > 2 else 0, n_as, size=(T, k)).astype(np.int32)
    if T > 40:
        ids[: T // 2, 0] = n_as - 1                      # one crowded group
    adapter = rng.integers(-1, n_adapters, size=T).astype(np.int32) if n_adapters else None
    want = group_ref(ids, n_as, adapter, n_adapters)
    wide = torch.from_numpy(np.concatenate([ids, np.full((T, 3), 77, np.int32)], 1)).cuda()
    for t in (torch.from_numpy(ids).cuda(), wide[:, :k]):           # packed rows, and rows of a wider tensor
        order, offsets = gxlib.group_rows(t, n_as, adapter=None if adapter is None else torch.from_numpy(adapter).cuda(),
                                          n_adapters=n_adapters)
        np.testing.assert_array_equal(offsets.cpu().numpy(), want[1])
        np.testing.assert_array_equal(order.cpu().numpy(), want[0])


def test_group_rows_adapters_alone_and_no_rows(gxlib, dev):
    a = np.array([2, -1, 0, 2, 1, 0, -1, 2], np.int32)
    order, offsets = gxlib.group_rows(None, adapter=torch.from_numpy(a).cuda(), n_adapters=4)
    assert order.tolist() == [2, 5, 4, 0, 3, 7, 1, 6] and offsets.tolist() == [0, 2, 3, 6, 6]
    order, offsets = gxlib.group_rows(torch.empty((0, 8), dtype=torch.int32, device="cuda"), 5)
    assert order.shape == (0,) and offsets.tolist() == [0] * 6
    order, offsets = gxlib.group_rows(torch.full((9, 4), -1, dtype=torch.int32, device="cuda"), 3)
    assert order.tolist() == list(range(36)) and offsets.tolist() == [0] * 4


def test_group_rows_reports_ids_outside_the_experts(gxlib, dev):
    from galactus_b200.moe import device_error
    device_error()
    order, offsets = gxlib.group_rows(torch.tensor([[0, 5], [4, 1]], dtype=torch.int32, device="cuda"), 5)
    assert order.tolist() == [0, 3, 2, 1] and offsets.tolist() == [0, 1, 2, 2, 2, 3]
    assert device_error() == 1 and device_error() == 0


# ------------------------------------------------------------------ products
def reference(w, x, counts, first, gather, order, scatter, n_rows, act=None, up=None, alpha=1.702, limit=7.0):
    """float64 results and error bounds (before the final rounding) of every row, NaN where no group has it."""
    N, K = w.shape[1], w.shape[2]
    out = torch.full((n_rows, N), float("nan"), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    j = first
    for g, c in enumerate(counts):
        if c:
            rows = torch.arange(j, j + c, device="cuda")
            src = order[rows].long() // gather if gather else rows
            xs = x[src].double()

            def dot(m):
                return xs @ m.double().T, (xs.abs() @ m.double().abs().T) * acc_bound(K)
            v, e = dot(w[g])
            if up is not None:
                u, eu = dot(up[g])
                if act == 1:
                    v, u, a = torch.clamp(v, max=limit), torch.clamp(u, -limit, limit) , alpha
                    u1 = u + 1.0
                else:
                    a, u1 = 1.0, u
                silu = v * torch.sigmoid(a * v)
                # |d(v sigmoid(a v))/dv| <= 1.1; exp, divide and products: 8 roundings of f32
                e = 1.1 * u1.abs() * e + silu.abs() * eu + 1.1 * e * eu + 8 * 2.0 ** -24 * (silu * u1).abs() \
                    + 4 * 2.0 ** -24 * silu.abs()
                v = silu * u1
            dst = order[rows].long() if scatter else rows
            out[dst], tol[dst] = v, e
        j += c
    return out, tol


def compare(got, want, tol, kind):
    got = got.double()
    err = (got - want).abs()
    lim = tol + HALF[kind] * (want.abs() + tol) + (2.0 ** -25 if kind == "f16" else 0.0)   # f16: half the subnormal step
    bad = ~(err <= lim)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / lim).max()):.3g} of the bound"


COUNTS = {
    "one": [1], "token": [0, 0, 1, 0, 1, 1, 0, 0, 1], "edges": [15, 16, 17, 0, 31, 32, 33, 0],
    "tiles": [127, 128, 129, 0, 1], "long": [0, 300, 0, 2, 513], "many": [1, 3, 0, 2] * 40, "none": [0, 0, 0],
    "few": [1, 0, 2, 1, 1], "middle": [40, 90, 0, 20, 64], "wide": [30, 5, 40, 61],
}


def make(G, K, N, rows, kind, seed, sigma=0.05, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = torch.randn((G, N, K + pad), generator=g, device="cuda").mul_(sigma).to(TYPES[kind])
    x = torch.randn((max(1, rows), K + pad), generator=g, device="cuda").to(TYPES[kind])
    return wide[:, :, :K], x[:rows, :K]


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("counts,K,N,kind,out", [
    ("one", 8, 1, "bf16", "f32"), ("one", 2048, 768, "f16", "f32"), ("token", 2880, 300, "f16", "f16"),
    ("edges", 72, 129, "bf16", "bf16"), ("edges", 1000, 63, "f16", "f32"), ("tiles", 64, 128, "bf16", "f32"),
    ("tiles", 520, 1001, "f16", "f16"), ("long", 256, 200, "bf16", "bf16"), ("many", 136, 257, "bf16", "f32"),
    ("none", 64, 64, "f16", "f32"), ("long", 4096, 384, "bf16", "f32"),
    # whole tiles for every SM and a rest that clusters share along K; one round of shared tiles
    ("few", 2880, 2880, "f16", "f16"), ("few", 2000, 2880, "bf16", "f32"), ("one", 7168, 64, "bf16", "f32"),
    # 64 and 128 rows a tile in single CTAs, several accumulators for f32 results
    ("middle", 1544, 500, "bf16", "f32"), ("wide", 328, 260, "f16", "bf16"), ("long", 512, 300, "f16", "f32"),
])
def test_products(gxlib, dev, counts, K, N, kind, out, glu):
    c = COUNTS[counts]
    P = sum(c)
    w, x = make(len(c), K, N, P, kind, K + N)
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(c)]), dtype=torch.int32, device="cuda")
    kw = dict(out_dtype=TYPES[out])
    if glu:
        up, _ = make(len(c), K, N, 0, kind, K + N + 1)
        act = K % 3 != 0
        got = gxlib.mul_mat_grouped_glu(w, up, x, offsets, act=int(act), **kw)
        want, tol = reference(w, x, c, 0, 0, None, False, P, int(act), up)
    else:
        got = gxlib.mul_mat_grouped(w, x, offsets, **kw)
        want, tol = reference(w, x, c, 0, 0, None, False, P)
    assert got.shape == (P, N) and got.dtype == TYPES[out]
    compare(got, want, tol, out)


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("T,k,E,gather,scatter", [(1, 4, 16, True, False), (1, 4, 16, False, True), (37, 3, 9, True, True),
                                                  (200, 8, 12, True, False), (333, 2, 5, False, True)])
def test_gather_scatter_and_foreign_rows(gxlib, dev, T, k, E, gather, scatter, glu):
    """Rows through the order of gx_group_rows, pairs without an expert among
    them, padded row strides everywhere, guard rows and columns left alone."""
    from galactus_b200.moe import device_error
    rng = np.random.default_rng(T)
    K, N, P = 200, 140, T * k
    ids = rng.integers(-1, E, size=(T, k)).astype(np.int32)
    order, offsets = gxlib.group_rows(torch.from_numpy(ids).cuda(), E)
    c = np.diff(offsets.cpu().numpy()).tolist()
    w, x = make(E, K, N, T if gather else P, "bf16", T + k, pad=8)
    up, _ = make(E, K, N, 0, "bf16", T + k + 1, pad=8)
    out = torch.full((P + 2, N + 6), 7.0, device="cuda")
    view = out[1:P + 1, 3:N + 3]
    kw = dict(order=order, gather=k if gather else 0, scatter=scatter, out=view)
    device_error()
    for again in range(2):
        if glu:
            gxlib.mul_mat_grouped_glu(w, up, x, offsets, **kw)
        else:
            gxlib.mul_mat_grouped(w, x, offsets, **kw)
        first = out.clone() if again == 0 else first
    assert torch.equal(out, first)                                   # the same bits again
    want, tol = reference(w, x, c, 0, k if gather else 0, order, scatter, P, 0 if glu else None, up if glu else None)
    kept = torch.isnan(want[:, 0])
    assert int(kept.sum()) == int((ids < 0).sum())
    assert bool((view[kept] == 7.0).all())
    compare(view[~kept], want[~kept], tol[~kept], "f32")
    out[1:P + 1, 3:N + 3] = 7.0
    assert bool((out == 7.0).all())                                  # nothing outside the rows was written
    assert device_error() == 0


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("K", [64, 1024])
def test_uneven_groups_gathered(gxlib, dev, K, glu):
    """Long and tiny groups side by side, many tiles per CTA: copying warps that have no rows in a tile keep step."""
    from galactus_b200.moe import device_error
    rng = np.random.default_rng(K)
    c = [700, 3, 256, 33, 1, 130, 0, 65, 31, 400, 2, 2] * 6
    E, N, P = len(c), 700, sum(c)
    order = torch.from_numpy(rng.permutation(P).astype(np.int32)).cuda()
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(c)]), dtype=torch.int32, device="cuda")
    w, x = make(E, K, N, P, "bf16", K)
    up, _ = make(E, K, N, 0, "bf16", K + 1)
    device_error()
    if glu:
        got = gxlib.mul_mat_grouped_glu(w, up, x, offsets, order=order, gather=1)
    else:
        got = gxlib.mul_mat_grouped(w, x, offsets, order=order, gather=1)
    assert device_error() == 0
    want, tol = reference(w, x, c, 0, 1, order, False, P, 0 if glu else None, up if glu else None)
    compare(got, want, tol, "bf16")


def test_first_border_above_zero_and_experts_in_a_record(gxlib, dev):
    """Matrices inside larger records (an arena's slots), rows in front of the first group."""
    K, N, c = 128, 96, [3, 0, 40]
    rec = torch.randn((3, 3 * N * K + 64), device="cuda").to(torch.float16)
    w = rec.as_strided((3, N, K), (rec.stride(0), K, 1), 64)
    x = torch.randn((50, K), device="cuda").to(torch.float16)
    offsets = torch.tensor([5, 8, 8, 48], dtype=torch.int32, device="cuda")
    out = torch.full((50, N), 3.0, dtype=torch.float16, device="cuda")
    gxlib.mul_mat_grouped(w, x, offsets, out=out)
    want, tol = reference(w, x, c, 5, 0, None, False, 50)
    assert bool((out[:5] == 3.0).all()) and bool((out[48:] == 3.0).all())
    compare(out[5:48], want[5:48], tol[5:48], "f16")


def test_nan_and_inf_stay_in_their_rows(gxlib, dev):
    K, N = 192, 130
    w, x = make(2, K, N, 40, "bf16", 5)
    x[7, 3], x[21, 100] = float("nan"), float("inf")
    offsets = torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda")
    got = gxlib.mul_mat_grouped(w, x, offsets, out_dtype=torch.float32)
    clean = x.clone()
    clean[7], clean[21] = 0, 0
    want, tol = reference(w, clean, [20, 20], 0, 0, None, False, 40)
    rows = [i for i in range(40) if i not in (7, 21)]
    compare(got[rows], want[rows], tol[rows], "f32")
    assert bool(torch.isnan(got[7]).all()) and not bool(torch.isfinite(got[21]).any())


def test_bad_borders_and_rows_are_reported(gxlib, dev):
    from galactus_b200.moe import device_error
    device_error()
    w, x = make(3, 64, 32, 10, "f16", 9)
    out = torch.full((10, 32), 5.0, device="cuda")
    good = gxlib.mul_mat_grouped(w, x, torch.tensor([0, 4, 4, 10], dtype=torch.int32, device="cuda"), out_dtype=torch.float32)
    gxlib.mul_mat_grouped(w, x, torch.tensor([0, 4, 2, 11], dtype=torch.int32, device="cuda"), out=out)
    assert torch.equal(out[:4], good[:4]) and bool((out[4:] == 5.0).all()) and device_error() == 1
    order = torch.tensor([0, 1, 2, 20, -1, 5, 6, 7, 8, 9], dtype=torch.int32, device="cuda")
    got = gxlib.mul_mat_grouped(w, x, torch.tensor([0, 10, 10, 10], dtype=torch.int32, device="cuda"), order=order, gather=1,
                                out_dtype=torch.float32)
    assert torch.isnan(got).all(1).tolist() == [i in (3, 4) for i in range(10)] and device_error() == 1
    out.fill_(5.0)
    gxlib.mul_mat_grouped(w, x, torch.tensor([0, 10, 10, 10], dtype=torch.int32, device="cuda"), order=order, scatter=True, out=out)
    assert (out == 5.0).all(1).tolist() == [i in (3, 4) for i in range(10)] and device_error() == 1


@pytest.mark.parametrize("K,N,kind,out", [(1, 1, "f16", "f32"), (3, 5, "bf16", "bf16"), (65, 130, "bf16", "f32"), (1001, 64, "f16", "f16")])
@pytest.mark.parametrize("glu", [False, True])
def test_lengths_that_are_no_multiple_of_anything(gxlib, dev, K, N, kind, out, glu):
    """Rows padded to 16 bytes; what lies in the padding is not read as numbers."""
    c = [3, 0, 20, 1]
    pad = -K % 8
    w, x = make(4, K, N, 24, kind, K, pad=pad)
    up, _ = make(4, K, N, 0, kind, K + 1, pad=pad)
    for t in (w, x, up):
        if pad:
            torch.as_strided(t, (*t.shape[:-1], pad), t.stride(), t.storage_offset() + K).fill_(float("nan"))
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(c)]), dtype=torch.int32, device="cuda")
    order = torch.arange(23, -1, -1, dtype=torch.int32, device="cuda")
    for gather in (0, 1):
        kw = dict(order=order, gather=gather, out_dtype=TYPES[out])
        got = gxlib.mul_mat_grouped_glu(w, up, x, offsets, **kw) if glu else gxlib.mul_mat_grouped(w, x, offsets, **kw)
        want, tol = reference(w, x, c, 0, gather, order, False, 24, 0 if glu else None, up if glu else None)
        compare(got, want, tol, out)


def test_thousands_of_groups_and_no_rows(gxlib, dev):
    E, K, N = 8192, 16, 24
    rng = np.random.default_rng(0)
    c = rng.integers(0, 3, size=E).tolist()
    P = sum(c)
    w, x = make(E, K, N, P, "bf16", 1)
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(c)]), dtype=torch.int32, device="cuda")
    got = gxlib.mul_mat_grouped(w, x, offsets, out_dtype=torch.float32)
    which = torch.repeat_interleave(torch.arange(E, device="cuda"), torch.tensor(c, device="cuda"))
    want = torch.einsum("pnk,pk->pn", w[which].double(), x.double())
    tol = torch.einsum("pnk,pk->pn", w[which].double().abs(), x.double().abs()) * acc_bound(K)
    compare(got, want, tol, "f32")
    zero = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert gxlib.mul_mat_grouped(w, x[:0], zero, order=none, scatter=True).shape == (0, N)
    assert gxlib.mul_mat_grouped_glu(w, w, x[:0], zero, order=none, gather=2).shape == (0, N)
    assert gxlib.lora_mul_mat(w, w.transpose(1, 2).contiguous(), x[:0], zero, base=torch.empty((0, K), device="cuda")).shape == (0, K)


def test_results_beyond_four_gigabytes(gxlib, dev):
    """Row 69999 of results that lie 65536 bytes apart, and deltas on such a base."""
    K, N, rows = 64, 64, 70000
    w, x = make(2, K, N, rows, "bf16", 2)
    wide = torch.zeros((rows, 16384), device="cuda")
    out = wide[:, -N:]
    offsets = torch.tensor([0, 100, rows], dtype=torch.int32, device="cuda")
    gxlib.mul_mat_grouped(w, x, offsets, out=out)
    want, tol = reference(w, x, [100, rows - 100], 0, 0, None, False, rows)
    compare(out, want, tol, "f32")
    a, b = make(2, K, 16, 0, "bf16", 3)[0], make(2, 16, N, 0, "bf16", 4)[0]
    before = out[-200:].clone()
    small = gxlib.lora_mul_mat(a[1:], b[1:], x[-200:], torch.tensor([0, 200], dtype=torch.int32, device="cuda"), base=before)
    gxlib.lora_mul_mat(a, b, x, offsets, base=out, out=out)
    # the sums of K and of the ranks may be split differently: f32 accuracy, not the same bits
    assert float((out[-200:] - small).abs().max()) <= 1e-5 * float(small.abs().max())
    assert bool((wide[:, :16384 - N] == 0).all())


def test_first_call_of_a_process_inside_a_capture(gxlib, dev):
    """Nothing has to be called before a capture: the first calls of a process may be captured ones."""
    import subprocess
    import sys
    code = """
import torch, galactus_b200 as gx
E, K, N, T, k = 6, 256, 200, 20, 2
g = torch.Generator(device="cuda").manual_seed(1)
w = torch.randn((E, N, K), device="cuda", generator=g).bfloat16()
x = torch.randn((T, K), device="cuda", generator=g).bfloat16()
a = torch.randn((E, 16, K), device="cuda", generator=g).bfloat16()
b = torch.randn((E, N, 16), device="cuda", generator=g).bfloat16()
ids = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
def layer():
    order, offsets = gx.group_rows(ids, E)
    y = gx.mul_mat_grouped(w, x, offsets, order=order, gather=k, scatter=True, out_dtype=torch.float32)
    h = gx.mul_mat_grouped_glu(w, w, x, offsets, order=order, gather=k)
    return gx.lora_mul_mat(a, b, x, offsets, order=order, gather=k, base=y), h
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = layer()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(got, layer()))
print("captured")
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=str(gxlib._lib.LIB_PATH.parent.parent))
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_calls_on_two_streams_at_once(gxlib, dev):
    """Nothing is shared between calls: products, grouping and deltas in flight together give the bits of calls alone."""
    E, K, N, T, k = 16, 1024, 512, 700, 4
    w, x = make(E, K, N, T, "bf16", 21)
    up, _ = make(E, K, N, 0, "bf16", 22)
    a, b = make(E, K, 16, 0, "bf16", 23)[0], make(E, 16, N, 0, "bf16", 24)[0]
    ids = torch.randint(0, E, (T, k), dtype=torch.int32, device="cuda")

    def work():
        order, offsets = gxlib.group_rows(ids, E)
        y = gxlib.mul_mat_grouped(w, x, offsets, order=order, gather=k, scatter=True, out_dtype=torch.float32)
        return gxlib.mul_mat_grouped_glu(w, up, x, offsets, order=order, gather=k), \
            gxlib.lora_mul_mat(a, b, x, offsets, order=order, gather=k, base=y, out=y)
    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g[0], want[0]) and torch.equal(g[1], want[1])


def test_capture_streams_and_wrapper_checks(gxlib, dev):
    K, N, T, k, E = 256, 192, 24, 2, 6
    w, x = make(E, K, N, T, "bf16", 3)
    up, _ = make(E, K, N, 0, "bf16", 4)
    ids = torch.randint(0, E, (T, k), dtype=torch.int32, device="cuda")

    def layer():
        order, offsets = gxlib.group_rows(ids, E)
        h = gxlib.mul_mat_grouped_glu(w, up, x, offsets, order=order, gather=k)
        return h
    want = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = layer()
    torch.cuda.synchronize()
    assert torch.equal(on_side, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer()
    ids.copy_((ids + 1) % E)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, layer())
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    for bad in (lambda: gxlib.mul_mat_grouped(w, x.half(), offsets), lambda: gxlib.mul_mat_grouped(w, x[:, :128], offsets),
                lambda: gxlib.mul_mat_grouped(w, x, offsets[:-1]), lambda: gxlib.mul_mat_grouped(w, x, offsets.long()),
                lambda: gxlib.mul_mat_grouped(w, x, offsets.cpu()), lambda: gxlib.mul_mat_grouped(w.transpose(1, 2), x, offsets),
                lambda: gxlib.mul_mat_grouped(w, x, offsets, out_dtype=torch.int32),
                lambda: gxlib.mul_mat_grouped_glu(w, up[:, :64], x, offsets)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(gxlib.GxError):
        gxlib.mul_mat_grouped(w, x, offsets, gather=2)               # an order is needed


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_round_rows(gxlib, dev, kind):
    x = torch.randn((5, 1030), device="cuda") * torch.logspace(-9, 6, 1030, device="cuda")
    x[1, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), -0.0], device="cuda")
    got = gxlib.round_rows(x[:, :1029], TYPES[kind])
    assert torch.equal(got.view(torch.int16)[:, 4:], x[:, :1029].to(TYPES[kind]).view(torch.int16)[:, 4:])
    assert torch.equal(torch.isnan(got), torch.isnan(x[:, :1029])) and got[1, 0] == float("inf") and got[1, 1] == -float("inf")


def test_unquantised_layer_from_an_arena(gxlib, dev):
    """The layer as it is used: router logits to ids, experts served into the
    slots of an arena, rows grouped by slot, gate/up and down read in place
    from the slab, combined in slot order."""
    from galactus_b200 import _lib as L
    from galactus_b200 import moe
    from galactus_b200.models import ModelShape
    H, I, E, k, T = 256, 192, 10, 3, 21
    m = ModelShape("f16-experts", 1, H, E, k, I, L.TYPE_F16, L.TYPE_F16, L.TYPE_F16)
    assert m.record_raw == 3 * H * I * 2
    rng = np.random.default_rng(0)
    recs = (rng.standard_normal((E, 3 * H * I)) * 0.06).astype(np.float16)
    arena = gxlib.Arena(m, capacity_bytes=E * m.record, policy=gxlib.POLICY_AUTO, max_tokens=T)
    try:
        for e in range(E):
            arena.load_record(0, e, recs[e].view(np.uint8))
        stream = torch.cuda.current_stream()
        arena.warm_all(stream)
        base, record, slots = arena.layer_view(0)
        desc = moe.router_desc(L.GX_GATING_SOFTMAX, E, k, norm_w=True)
        logits = torch.randn((T, E), device="cuda")
        table = moe.slot_table(arena, 0, 1)
        sl = torch.empty((T, k), dtype=torch.int32, device="cuda")
        ids, wts = moe.route(desc, logits, slot_table=table, slots=sl)
        x = torch.randn((T, H), device="cuda")
        xr = gxlib.round_rows(x, torch.float16)
        order, offsets = gxlib.group_rows(sl, slots)
        lib, s = gxlib.lib(), stream.cuda_stream
        h = torch.empty((T * k, I), dtype=torch.float16, device="cuda")
        gxlib.check(lib.gx_mul_mat_grouped_glu(L.TYPE_F16, base + m.off_gate, base + m.off_up, H, I, 2 * H, record, slots,
                                               xr.data_ptr(), T, 2 * H, offsets.data_ptr(), order.data_ptr(), T * k, k, 0, 0,
                                               0.0, 0.0, L.TYPE_F16, h.data_ptr(), 2 * I, s))
        y = torch.empty((T, k, H), device="cuda")
        gxlib.check(lib.gx_mul_mat_grouped(L.TYPE_F16, base, I, H, 2 * I, record, slots, h.data_ptr(), T * k, 2 * I,
                                           offsets.data_ptr(), order.data_ptr(), T * k, 0, 1, L.TYPE_F32, y.data_ptr(), 4 * H, s))
        out = torch.empty((T, H), device="cuda")
        gxlib.check(lib.gx_combine(y.data_ptr(), wts.data_ptr(), out.data_ptr(), H, k, T, s))
        torch.cuda.synchronize()
        down = torch.from_numpy(recs[:, :H * I].reshape(E, H, I)).cuda().double()
        gate = torch.from_numpy(recs[:, H * I:2 * H * I].reshape(E, I, H)).cuda().double()
        upm = torch.from_numpy(recs[:, 2 * H * I:].reshape(E, I, H)).cuda().double()
        want = torch.zeros((T, H), dtype=torch.float64, device="cuda")
        lim = torch.zeros_like(want)
        for t in range(T):
            for j in range(k):
                e = int(ids[t, j])
                xe = xr[t].double()
                g, u = gate[e] @ xe, upm[e] @ xe
                a = g * torch.sigmoid(g) * u
                # the f16 rounding of the activation, and f32 sums far below it
                ea = a.abs() * (HALF["f16"] + 2.0 ** -18) + 1.1 * (u.abs() + g.abs()) * (gate[e].abs() @ xe.abs()) * acc_bound(H) \
                    + (1.1 * u.abs() + g.abs()) * (upm[e].abs() @ xe.abs()) * acc_bound(H) + 2.0 ** -25
                wt = float(wts[t, j])
                want[t] += wt * (down[e] @ a)
                lim[t] += wt * (down[e].abs() @ ea + (down[e].abs() @ a.abs()) * (acc_bound(I) + 4 * 2.0 ** -24))
        assert bool(((out.double() - want).abs() <= lim).all())
    finally:
        arena.close()
