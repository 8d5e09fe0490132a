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
