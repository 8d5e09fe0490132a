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
