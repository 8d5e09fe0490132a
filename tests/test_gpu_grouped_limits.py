"""The operators on grouped rows at the ends of what they accept: the largest
group counts and ranks, long sums, several host threads, other streams."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_lora import compare, keys_of, make, reference  # noqa: E402


@pytest.mark.parametrize("n_as,adapters,rank,K", [(41, 199, 100, 16), (128, 64, 128, 520), (1, 8192, 65, 72)])
def test_adapters_at_the_largest_group_counts(gxlib, dev, n_as, adapters, rank, K):
    """Ranks above 64 and 8159 to 8192 groups leave room for two stages of the ring, the fewest it works with."""
    from galactus_b200.moe import device_error
    device_error()
    T, k, N = 301, 2 if n_as > 1 else 1, 24
    rng = np.random.default_rng(adapters)
    s = make(T, k, n_as, adapters, rank, K, N, "bf16", "f32", adapters)
    ids = rng.integers(0, n_as, size=(T, k)).astype(np.int32)
    adapter = rng.integers(-1, adapters, size=T).astype(np.int32)
    adapter[:70], ids[:70] = adapters - 1, n_as - 1                  # the last group, more than a tile of it
    ranks = rng.integers(0, rank + 1, size=adapters).astype(np.int32)
    ranks[-1] = rank
    order, offsets = gxlib.group_rows(torch.from_numpy(ids).cuda() if n_as > 1 else None, n_as,
                                      adapter=torch.from_numpy(adapter).cuda(), n_adapters=adapters)
    want, tol = reference(s, keys_of(ids, adapter, n_as), k, n_as, ranks, np.ones(adapters))
    got = gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, order=order, gather=k, n_as=n_as, base=s["base"],
                             ranks=torch.from_numpy(ranks).cuda())
    compare(got, want, tol, "f32")
    assert device_error() == 0


@pytest.mark.parametrize("T,K,N,rank,adapters", [(1, 4096, 64, 16, 1), (40, 7168, 130, 64, 9), (300, 2048, 1, 16, 40), (5, 64, 1000, 128, 5)])
def test_adapters_with_ctas_that_have_no_share(gxlib, dev, T, K, N, rank, adapters):
    """Clusters of more CTAs than result tiles or chunks of K, call after call: each CTA leaves with its barriers at rest."""
    from galactus_b200.moe import device_error
    device_error()
    s = make(T, 1, 1, adapters, rank, K, N, "f16", "f32", T)
    adapter = np.random.default_rng(T).integers(-1 if T > 2 else 0, adapters, size=T).astype(np.int32)
    order, offsets = gxlib.group_rows(None, adapter=torch.from_numpy(adapter).cuda(), n_adapters=adapters)
    want, tol = reference(s, adapter.astype(np.int64), 1, 1, [rank] * adapters, [1.0] * adapters)
    first = gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, order=order, base=s["base"])
    compare(first, want, tol, "f32")
    got = [gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, order=order, base=s["base"]) for _ in range(50)]
    assert all(torch.equal(g, first) for g in got)
    assert device_error() == 0


def test_host_threads_with_calls_of_different_sizes(gxlib, dev):
    """Every kernel's shared memory differs from call to call; threads that call at once do not get in each other's way."""
    import threading
    g = torch.Generator(device="cuda").manual_seed(3)

    def job(E, K, N, rank, T):
        rnd = lambda *s: (torch.randn(s, generator=g, device="cuda") * 0.1).bfloat16()
        w, up, x, a, b = rnd(E, N, K), rnd(E, N, K), rnd(T, K), rnd(E, rank, K), rnd(E, N, rank)
        ids = torch.randint(0, E, (T, 1), generator=g, device="cuda", dtype=torch.int32)
        base = torch.randn((T, N), generator=g, device="cuda")

        def run():
            order, offsets = gxlib.group_rows(ids, E)
            return (order, offsets, gxlib.mul_mat_grouped(w, x, offsets, order=order, gather=1, out_dtype=torch.float32),
                    gxlib.mul_mat_grouped_glu(w, up, x, offsets, order=order, gather=1),
                    gxlib.lora_mul_mat(a, b, x, offsets, order=order, base=base))
        return run
    jobs = [job(*a) for a in ((2, 64, 32, 16, 5), (4096, 64, 32, 128, 40), (300, 512, 64, 64, 9), (1, 256, 130, 32, 700))]
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    failed, gate = [], threading.Barrier(len(jobs))

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait()
                for _ in range(150):
                    got = jobs[i]()
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(p, q) for p, q in zip(got, want[i])):
                failed.append((i, "other results"))
        except Exception as e:                                       # noqa: BLE001
            failed.append((i, repr(e)))
            gate.abort()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_a_graph_keeps_its_large_call_after_a_small_one(gxlib, dev):
    """A captured call of many groups and one of few share their kernel; replays and calls in between keep their sizes."""
    def inputs(E, T):
        ids = torch.randint(0, E, (T, 1), device="cuda", dtype=torch.int32)
        return ids, (torch.randn((E, 40, 64), device="cuda") * 0.1).half(), torch.randn((T, 64), device="cuda").half(), E

    def run(ids, w, x, E):
        order, offsets = gxlib.group_rows(ids, E)
        return gxlib.mul_mat_grouped(w, x, offsets, order=order, gather=1, out_dtype=torch.float32)
    large, small = inputs(8192, 100), inputs(3, 7)
    want = run(*large), run(*small)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*large), run(*small)
    for _ in range(3):
        for t in got:
            t.zero_()
        run(*small)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("handle", [False, True])
def test_results_allocated_for_another_stream(gxlib, dev, handle):
    """A result allocated by a call on `stream` takes no memory that work queued on the current stream still reads."""
    E, K, N, T = 5, 256, 512, 3000
    w, up, a, b = ((torch.randn(s, device="cuda") * 0.1).bfloat16() for s in ((E, N, K), (E, N, K), (E, 16, K), (E, N, 16)))
    x32, base = torch.randn((T, K), device="cuda"), torch.randn((T, N), device="cuda")
    x = x32.bfloat16()
    ids = torch.randint(0, E, (200000, 1), device="cuda", dtype=torch.int32)
    order, offsets = gxlib.group_rows(ids[:T], E)
    side = torch.cuda.Stream()
    calls = [
        lambda s: gxlib.group_rows(ids, E, stream=s)[0],
        lambda s: gxlib.round_rows(x32, torch.bfloat16, stream=s),
        lambda s: gxlib.mul_mat_grouped(w, x, offsets, order=order, gather=1, out_dtype=torch.float32, stream=s),
        lambda s: gxlib.mul_mat_grouped_glu(w, up, x, offsets, order=order, gather=1, stream=s),
        lambda s: gxlib.lora_mul_mat(a, b, x, offsets, order=order, base=base, stream=s),
    ]
    for call in calls:
        want = call(None)
        sink = torch.empty_like(want)
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        read = torch.full_like(want, 3)
        torch.cuda.synchronize()
        torch.cuda._sleep(100_000_000)                              # about 50 ms: `read` is given back with its reader still queued
        sink.copy_(read)
        del read
        got = call(side.cuda_stream if handle else side)
        side.synchronize()
        assert torch.equal(got, want)
        torch.cuda.synchronize()
        assert bool((sink == 3).all())
    with torch.cuda.stream(side):                                    # and the default stream while another is current
        got = calls[2](0 if handle else torch.cuda.default_stream())
        torch.cuda.synchronize()
        assert torch.equal(got, calls[2](None))


def long_bound(K: int) -> float:
    """Of an f32 sum of K products of one sign, relative to it, when an accumulator takes 512 of them: a step of an
    accumulator adds 16 products to a sum that is at most the whole (one step of it, 2^-23, and the alignment of the 16,
    as much each); then one rounded add per accumulator and per CTA that shares K (at most eight), 2^-24 each."""
    return (512 / 16 + 16) * 2.0 ** -23 + (K / 512 + 1 + 8) * 2.0 ** -24


def positive(shape, sigma, seed, kind="bf16"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda").abs_() * sigma).to({"bf16": torch.bfloat16, "f16": torch.float16}[kind])


@pytest.mark.parametrize("T,K,kind", [(6400, 28672, "bf16"), (6400, 7168, "f16"), (3, 28672, "bf16"), (700, 14336, "f16"), (5000, 3080, "bf16")])
def test_long_sums_of_adapters(gxlib, dev, T, K, kind):
    """Products of one sign, where a truncating sum shows as a bias: f32 results keep f32 accuracy however long K is,
    with one CTA per tile of rows (6400 rows) and with clusters."""
    N, rank = 64, 16
    x, a, b = positive((T, K), 1.0, 1, kind), positive((1, rank, K), 1.0 / K, 2, kind), positive((1, N, rank), 0.1, 3, kind)
    offsets = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    got = gxlib.lora_mul_mat(a, b, x, offsets, base=torch.zeros((T, N), device="cuda")).double()
    want = torch.cat([(c.double() @ a[0].double().T) @ b[0].double().T for c in x.split(1024)])
    # h, its parts (2^-22), 48 products of the second sum, the last add
    bound = long_bound(K) + 2.0 ** -22 + (48 / 16 + 16) * 2.0 ** -23 + 2.0 ** -24
    off = float(((got - want).abs() / want).max())
    assert off <= bound, f"{off:.3g} of {bound:.3g}"


@pytest.mark.parametrize("rows,N", [(300, 200), (3, 200), (40, 130), (3, 4096)])
@pytest.mark.parametrize("glu", [False, True])
def test_long_sums_of_products(gxlib, dev, rows, N, glu):
    """The same of the products: CTA pairs, single CTAs, and clusters that share K."""
    K = 28672
    x, w, up = positive((rows, K), 1.0, 4), positive((2, N, K), 1.0 / K, 5), positive((2, N, K), 2.0 / K, 6)
    offsets = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device="cuda")
    g = torch.cat([x[:rows // 3].double() @ w[0].double().T, x[rows // 3:].double() @ w[1].double().T])
    if glu:
        got = gxlib.mul_mat_grouped_glu(w, up, x, offsets, out_dtype=torch.float32)
        u = torch.cat([x[:rows // 3].double() @ up[0].double().T, x[rows // 3:].double() @ up[1].double().T])
        want = g * torch.sigmoid(g) * u
        # both sums (d silu(g) / dg * g <= 2 silu(g) for g > 0), eight roundings of the activation
        bound = 3 * long_bound(K) + 8 * 2.0 ** -23
    else:
        got = gxlib.mul_mat_grouped(w, x, offsets, out_dtype=torch.float32)
        want, bound = g, long_bound(K)
    off = float(((got.double() - want).abs() / want).max())
    assert off <= bound, f"{off:.3g} of {bound:.3g}"


def test_an_infinite_h_beside_large_ones_in_f16(gxlib, dev):
    """One rank's h is infinite, another's finite but beyond F16: the results are infinite with the first one's sign, not NaN."""
    T, K, N, rank = 20, 64, 200, 16
    x = positive((T, K), 1000.0, 1, "f16") + 1
    a = torch.zeros((1, rank, K), dtype=torch.float16, device="cuda")
    a[0, 0, 5], a[0, 1] = float("inf"), 1000.0
    a[0, 0, 6:] = 1.0
    a[0, 0, :5] = 1.0
    b = torch.zeros((1, N, rank), dtype=torch.float16, device="cuda") + 0.5
    b[0, ::2, 0] = -0.5
    b[0, :, 1] = -b[0, :, 0]
    offsets = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    # (the remaining ranks' h are zero: 0 * inf does not arise)
    got = gxlib.lora_mul_mat(a, b, x, offsets, base=torch.zeros((T, N), device="cuda"))
    want = torch.where(b[0, :, 0] > 0, float("inf"), float("-inf")).expand(T, N)
    assert torch.equal(got, want)


@pytest.mark.parametrize("size", [1e-34, 1e-30, 1e-20, 1e30])
def test_h_of_any_size_in_f16(gxlib, dev, size):
    """F16 adapters at the ends of f32: the row's power of two keeps at least 22 bits of h."""
    s = make(40, 1, 1, 1, 16, 128, 96, "f16", "f32", 12)
    s["base"].zero_()
    offsets = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    scale = torch.tensor([size], device="cuda")
    want, tol = reference(s, np.zeros(40, np.int64), 1, 1, [16], [float(scale[0])])
    got = gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, base=s["base"], scale=scale)
    # (below 2^-126 of the result, f32 itself ends)
    assert bool(((got.double() - want).abs() <= tol + 2.0 ** -23 * want.abs() + 2.0 ** -149).all())


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("kind,out", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_activation_over_the_whole_range(gxlib, dev, kind, out, act, rows):
    """The gated activation on exactly known gates and ups: a fine grid, the ends where e^-g leaves f32, infinities and
    NaN; single CTAs and pairs."""
    half = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[out]
    dtype = {"bf16": torch.bfloat16, "f16": torch.float16}[kind]
    alpha, limit = (1.702, 7.0) if act else (1.0, float("inf"))
    grid = np.concatenate([np.linspace(-95, 95, 1501), -np.linspace(50, 54, 300), -np.linspace(86.5, 89.5, 300),
                           [0.0, -0.0, 1e-3, -1e-3, 3e4, -3e4, np.inf, -np.inf, np.nan]])
    ups = np.array([1.0, -3.5, 0.0, 7.0, 2.0 ** 14, 2.0 ** -14] + ([2.0 ** 100] if kind == "bf16" else []) + [np.inf, np.nan])
    g0, u0 = (torch.from_numpy(v.reshape(-1)).cuda() for v in np.meshgrid(grid, ups))
    N = g0.numel()
    hi = g0.to(dtype)
    lo = torch.where(torch.isfinite(hi), g0 - hi.double(), torch.zeros_like(g0)).to(dtype)
    gate, up = (torch.zeros((1, N, 8), dtype=dtype, device="cuda") for _ in range(2))
    gate[0, :, 0], gate[0, :, 1], up[0, :, 2] = hi, lo, u0.to(dtype)
    x = torch.zeros((rows, 8), dtype=dtype, device="cuda")
    x[:, :3] = 1.0
    offsets = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    types = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
    got = gxlib.mul_mat_grouped_glu(gate, up, x, offsets, act=act, alpha=alpha, limit=limit if act else 7.0, out_dtype=types[out])
    assert torch.equal(got.view(torch.int16 if out != "f32" else torch.int32), got[:1].expand(rows, N).contiguous().view(
        torch.int16 if out != "f32" else torch.int32))
    got = got[0].double()
    g, u = hi.double() + lo.double(), up[0, :, 2].double()
    if act:
        g, u = torch.where(g > limit, limit, g), torch.where(u > limit, limit, torch.where(u < -limit, -limit, u)) + 1.0
    z = -float(np.float32(alpha)) * g
    e = torch.exp(z)
    e = torch.where(e >= 2.0 ** 128, float("inf"), e)                # (f32, as gx_swiglu: 1 / (1 + inf) is zero)
    want = g / (1.0 + e) * u
    # f32: e^z within 2 steps, 16 bits: CUDA's fast exp, 2 + 1.173 |z| steps; the product alpha * x moves e^z by |z| half
    # steps; the division 2 steps; the sum and the products (three, with u + 1) half a step each
    steps = (4.0 if out == "f32" else 4.0 + 2.35 * z.abs()) + (z.abs() if act else 0.0) + 4.0 + 4.0
    tol = torch.nan_to_num(steps * 2.0 ** -24 * want.abs(), nan=0.0, posinf=0.0)
    # and half a step of the type's smallest numbers: f16's is 2^-24, bf16's 2^-133, f32's 2^-149 (twice: the quotient's too)
    tol = tol + half * (want.abs() + tol) + {"f32": 2.0 ** -149, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}[out]
    top = {"f32": 3e38, "bf16": 3e38, "f16": 65000.0}[out]
    finite = torch.isfinite(want) & (want.abs() < top)
    bad = finite & ~((got - want).abs() <= tol)
    assert not bool(bad.any()), [(float(g[i]), float(u[i]), float(got[i]), float(want[i])) for i in bad.nonzero()[:5, 0].tolist()]
    wild = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got[wild]), torch.isnan(want[wild]))
    keep = wild & ~torch.isnan(want)
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("groups", [3, 8191])
def test_borders_that_overlap_many_times(gxlib, dev, groups):
    """0, n, 0, n, ...: more rows than there are. Every second group descends and is skipped; with many of the others,
    the tiles could outnumber what an index holds, and the call is dropped as a whole."""
    from galactus_b200.moe import device_error
    device_error()
    n, K, N = 40, 64, 32
    w = torch.randn((groups, N, K), device="cuda").half()
    a, b = torch.randn((groups, 16, K), device="cuda").half(), torch.randn((groups, N, 16), device="cuda").half()
    x = torch.randn((n, K), device="cuda").half()
    offsets = torch.tensor([0, n] * (groups // 2 + 1), dtype=torch.int32, device="cuda")[:groups + 1].contiguous()
    out = torch.full((n, N), 5.0, device="cuda")
    gxlib.mul_mat_grouped(w, x, offsets, out=out)
    assert device_error() == 1 and (groups == 3 or bool((out == 5.0).all()))
    out.fill_(5.0)
    gxlib.mul_mat_grouped_glu(w, w, x, offsets, out=out)
    assert device_error() == 1 and (groups == 3 or bool((out == 5.0).all()))
    out.fill_(5.0)
    gxlib.lora_mul_mat(a, b, x, offsets, base=torch.zeros_like(out), out=out)
    assert device_error() == 1 and (groups == 3 or bool((out == 5.0).all()))
    one = torch.tensor([0] + [n] * groups, dtype=torch.int32, device="cuda")     # and good borders work as before
    assert bool(torch.isfinite(gxlib.mul_mat_grouped(w, x, one, out_dtype=torch.float32)).all()) and device_error() == 0


@pytest.mark.parametrize("E,N,K", [(1, 40, 64), (4, 1, 64), (1, 1, 8)])
def test_gate_and_up_with_strides_that_nothing_uses(gxlib, dev, E, N, K):
    """One expert, or one row per expert: the strides that lead to no second one may differ."""
    gate = torch.randn((E, N, K), device="cuda").bfloat16()
    up = torch.randn((E, N, K), device="cuda").bfloat16()
    x = torch.randn((9, K), device="cuda").bfloat16()
    offsets = torch.tensor([0] * E + [9], dtype=torch.int32, device="cuda")
    wide = torch.zeros((E, N + 3, K), dtype=torch.bfloat16, device="cuda")
    wide[:, :N] = up
    other = wide[:, :N] if E == 1 else up.as_strided((E, N, K), (K, 5 * K, 1))
    assert other.stride() != gate.stride()
    assert torch.equal(gxlib.mul_mat_grouped_glu(gate, other, x, offsets), gxlib.mul_mat_grouped_glu(gate, up, x, offsets))
    if E == 1 and N > 1:
        with pytest.raises(ValueError):
            gxlib.mul_mat_grouped_glu(gate, torch.zeros((E, N, 2 * K), device="cuda").bfloat16()[:, :, :K], x, offsets)


def test_rounding_of_very_long_rows(gxlib, dev):
    """More columns than one CTA per 1024 of them can cover."""
    n = 65535 * 1024 + 70001
    x = torch.randn((2, n), device="cuda")
    assert torch.equal(gxlib.round_rows(x, torch.bfloat16), x.bfloat16())


def test_adapters_of_a_very_wide_projection(gxlib, dev):
    """Rows of base of more than a megabyte (an output head's)."""
    s = make(3, 1, 1, 1, 8, 64, 300001, "bf16", "f32", 2)
    want, tol = reference(s, np.zeros(3, np.int64), 1, 1, [8], [1.0])
    offsets = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    compare(gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, base=s["base"]), want, tol, "f32")
    wide = make(3, 1, 1, 1, 8, 64, 300032, "bf16", "f32", 3)
    want, tol = reference(wide, np.zeros(3, np.int64), 1, 1, [8], [1.0])
    compare(gxlib.lora_mul_mat(wide["a"], wide["b"], wide["x"], offsets, base=wide["base"]), want, tol, "f32")


@pytest.mark.parametrize("rows", [3, 300])
def test_very_long_sums_with_f16_results(gxlib, dev, rows):
    """Where a truncating sum would show beside the rounding of a 16-bit result, it is cut as well."""
    K, N = 1 << 17, 70
    x, w = positive((rows, K), 1.0, 1, "f16"), positive((1, N, K), 1.0 / 64, 2, "f16")
    scale = 2.0 ** -4                                                # (sums near 1000 in f16)
    w.mul_(scale)
    offsets = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    got = gxlib.mul_mat_grouped(w, x, offsets, out_dtype=torch.float16).double()
    want = x.double() @ w[0].double().T
    bound = long_bound(K) + 2.0 ** -11 * (1 + long_bound(K))
    off = float(((got - want).abs() / want).max())
    assert off <= bound, f"{off:.3g} of {bound:.3g}"
    a, b = positive((1, 16, K), 1.0 / K, 3, "f16"), positive((1, N, 16), 0.1, 4, "f16")
    a = torch.where(a > 2.0 ** -16, a, a + 2.0 ** -16)               # (normal and subnormal f16 alike, all of one sign)
    got = gxlib.lora_mul_mat(a, b, x, offsets, base=torch.zeros((rows, N), dtype=torch.float16, device="cuda")).double()
    want = (x.double() @ a[0].double().T) @ b[0].double().T
    bound = long_bound(K) + 2.0 ** -22 + (48 / 16 + 16) * 2.0 ** -23 + 2.0 ** -24
    bound += 2.0 ** -11 * (1 + bound)
    off = float(((got - want).abs() / want).max())
    assert off <= bound, f"{off:.3g} of {bound:.3g}"


@pytest.mark.parametrize("K,N,rank,kind,out", [(1, 1, 1, "f16", "f32"), (5, 3, 3, "bf16", "bf16"), (65, 130, 17, "bf16", "f32"), (131, 127, 33, "f16", "f16")])
def test_adapters_with_lengths_that_are_no_multiple(gxlib, dev, K, N, rank, kind, out):
    """Rows padded to 16 bytes, NaN in the padding; no order and two rows of base per row of x, then an order."""
    T, k = 21, 2
    s = make(T, k, 1, 3, rank, K, N, kind, out, K)

    def padded(t):
        wide = torch.full((*t.shape[:-1], (t.shape[-1] + 7) // 8 * 8 + 8), float("nan"), dtype=t.dtype, device="cuda")
        wide[..., :t.shape[-1]] = t
        return wide[..., :t.shape[-1]]
    a, b, x = padded(s["a"]), padded(s["b"]), padded(s["x"])
    offsets = torch.tensor([0, 5, 5, 39], dtype=torch.int32, device="cuda")
    keys = np.array([0] * 5 + [2] * 34 + [-1] * 3)
    want, tol = reference(s, keys, k, 1, [rank] * 3, [1.0] * 3)
    compare(gxlib.lora_mul_mat(a, b, x, offsets, gather=k, base=s["base"]), want, tol, out)
    order = torch.randperm(T * k, device="cuda").int()
    back = np.empty(T * k, np.int64)
    back[order.cpu().numpy()] = keys
    want, tol = reference(s, back, k, 1, [rank] * 3, [1.0] * 3)
    compare(gxlib.lora_mul_mat(a, b, x, offsets, order=order, gather=k, base=s["base"]), want, tol, out)


@pytest.mark.parametrize("rows", [1, 70, 5000])
def test_no_row_has_an_adapter(gxlib, dev, rows):
    """Every row is copied, bit for bit (NaN payloads too), or left alone in place; so with adapters of rank 0."""
    from galactus_b200.moe import device_error
    device_error()
    s = make(rows, 1, 1, 4, 16, 64, 100, "bf16", "f32", rows)
    s["base"].view(torch.int32)[:, 3] = 0x7fc12345
    none = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    some = torch.arange(rows, device="cuda").int() % 4
    for adapter, ranks in ((none, None), (some, torch.zeros(4, dtype=torch.int32, device="cuda"))):
        order, offsets = gxlib.group_rows(None, adapter=adapter, n_adapters=4)
        got = gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, order=order, ranks=ranks, base=s["base"])
        assert torch.equal(got.view(torch.int32), s["base"].view(torch.int32))
        here = s["base"].clone()
        gxlib.lora_mul_mat(s["a"], s["b"], s["x"], offsets, order=order, ranks=ranks, base=here, out=here)
        assert torch.equal(here.view(torch.int32), s["base"].view(torch.int32))
    assert device_error() == 0


def test_group_rows_of_millions_of_pairs_into_given_buffers(gxlib, dev):
    T, k, E = (1 << 20) + 13, 8, 200
    ids = torch.randint(-1, E, (T, k), dtype=torch.int32, device="cuda")
    order = torch.full((T * k,), -7, dtype=torch.int32, device="cuda")
    offsets = torch.full((E + 1,), -7, dtype=torch.int32, device="cuda")
    got = gxlib.group_rows(ids, E, order=order, offsets=offsets)
    assert got[0] is order and got[1] is offsets
    key, want = torch.sort(torch.where(ids < 0, E, ids).reshape(-1), stable=True)
    assert torch.equal(order, want.int())
    assert torch.equal(offsets, torch.searchsorted(key, torch.arange(E + 1, device="cuda", dtype=torch.int32)).int())


@pytest.mark.parametrize("rows", [6, 300])
def test_fewer_rows_than_the_order_holds(gxlib, dev, rows):
    """n_rows: the groups end before the order does; a result with more rows than that keeps the others."""
    K, N = 72, 40
    w, x = (torch.randn((3, N, K), device="cuda") * 0.1).bfloat16(), torch.randn((rows + 9, K), device="cuda").bfloat16()
    order = torch.randperm(rows + 9, device="cuda").int()
    offsets = torch.tensor([0, rows // 2, rows // 2, rows], dtype=torch.int32, device="cuda")
    out = torch.full((rows + 4, N), 7.0, device="cuda")
    got = gxlib.mul_mat_grouped(w, x, offsets, order=order, n_rows=rows, gather=1, out=out)
    assert got is out and bool((out[rows:] == 7.0).all())
    g = torch.cat([torch.zeros(rows // 2, dtype=torch.long), torch.full((rows - rows // 2,), 2)]).cuda()
    xs = x[order[:rows].long()].double()
    want = torch.einsum("jnk,jk->jn", w[g].double(), xs)
    tol = torch.einsum("jnk,jk->jn", w[g].double().abs(), xs.abs()) * (K / 16 + 16) * 2.0 ** -23
    compare(out[:rows], want, tol, "f32")
