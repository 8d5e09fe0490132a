"""Host-side checks of the operators on grouped rows: every refusal happens
before any device work, so it is the same with and without a GPU."""
import pytest

F32, F16, BF16 = 0, 1, 30
OK, INVALID, TYPE, ALIGN = 0, -1, -2, -3


def product(gxlib, **over):
    a = dict(type=BF16, w=4096, ne00=64, ne01=48, nb01=128, nb02=48 * 128, n_as=4, b=4096, ne11=10, nb11=128, offsets=4096,
             order=4096, n_rows=10, gather=0, scatter=0, type_dst=F32, dst=4096, nbd1=192)
    assert set(over) <= set(a)
    a.update(over)
    return gxlib.lib().gx_mul_mat_grouped(*a.values(), None)


def glu(gxlib, **over):
    a = dict(type=F16, gate=4096, up=8192, ne00=64, ne01=48, nb01=128, nb02=48 * 128, n_as=4, b=4096, ne11=10, nb11=128,
             offsets=4096, order=4096, n_rows=10, gather=0, scatter=0, act=0, alpha=1.702, limit=7.0, type_dst=F16, dst=4096,
             nbd1=96)
    assert set(over) <= set(a)
    a.update(over)
    return gxlib.lib().gx_mul_mat_grouped_glu(*a.values(), None)


COMMON = [
    (dict(type=F32), TYPE), (dict(type=8), TYPE), (dict(type_dst=8), TYPE),
    (dict(ne00=0), INVALID), (dict(ne01=0), INVALID), (dict(n_as=0), INVALID), (dict(n_as=8193), INVALID),
    (dict(n_rows=-1), INVALID), (dict(gather=-1), INVALID), (dict(scatter=2), INVALID),
    (dict(nb01=112), INVALID), (dict(nb11=112), INVALID), (dict(nbd1=64), INVALID), (dict(nb02=128), INVALID),
    (dict(nb01=1 << 40), INVALID), (dict(ne11=9), INVALID), (dict(ne11=0), INVALID),
    (dict(b=None), INVALID), (dict(offsets=None), INVALID), (dict(dst=None), INVALID),
    (dict(order=None, scatter=1), INVALID), (dict(order=None, gather=2), INVALID),
    (dict(nb01=136), ALIGN), (dict(nb11=136), ALIGN), (dict(nb02=48 * 128 + 8), ALIGN), (dict(b=4104), ALIGN),
    (dict(offsets=4098), ALIGN), (dict(order=4097), ALIGN), (dict(dst=4097), ALIGN),
    (dict(n_rows=0, b=None, dst=None, order=None, offsets=None, ne11=0), OK),
    (dict(ne01=1 << 30, nb01=1 << 39, nb02=1 << 39, nbd1=1 << 33), INVALID),      # a matrix of 2^69 bytes
]


@pytest.mark.parametrize("over,want", COMMON + [(dict(w=None), INVALID), (dict(w=4104), ALIGN), (dict(nbd1=194), ALIGN)])
def test_product_refusals(gxlib, over, want):
    assert product(gxlib, **over) == want


@pytest.mark.parametrize("over,want", COMMON + [(dict(gate=None), INVALID), (dict(up=None), INVALID), (dict(up=8200), ALIGN),
                                                (dict(act=2), INVALID), (dict(nbd1=97), ALIGN)])
def test_glu_refusals(gxlib, over, want):
    assert glu(gxlib, **over) == want


@pytest.mark.parametrize("over,want", [
    (dict(k=0), INVALID), (dict(T=-1), INVALID), (dict(n_as=0), INVALID), (dict(n_adapters=-1), INVALID),
    (dict(ids=None), INVALID), (dict(order=None), INVALID), (dict(offsets=None), INVALID),
    (dict(n_adapters=2), INVALID), (dict(adapter=4096), INVALID),
    (dict(ids=None, adapter=4096, n_adapters=2), INVALID),          # two slots a token, but no ids
    (dict(n_as=8193), INVALID), (dict(n_as=128, adapter=4096, n_adapters=65), INVALID),
    (dict(nbi1=4), INVALID), (dict(nbi1=10), INVALID), (dict(T=1 << 30), INVALID),
    (dict(ids=4098), ALIGN), (dict(order=4097), ALIGN), (dict(offsets=4099), ALIGN),
])
def test_group_refusals(gxlib, over, want):
    a = dict(ids=4096, k=2, T=5, nbi1=8, adapter=None, n_as=64, n_adapters=0, order=4096, offsets=4096)
    a.update(over)
    assert gxlib.lib().gx_group_rows(*a.values(), None) == want


@pytest.mark.parametrize("args,want", [
    ((F16, None, 8, 1, 32, 4096, 16), INVALID), ((BF16, 4096, 0, 1, 32, 4096, 16), INVALID),
    ((BF16, 4096, 8, -1, 32, 4096, 16), INVALID), ((BF16, 4096, 8, 1, 30, 4096, 16), INVALID),
    ((F16, 4096, 8, 1, 32, 4096, 14), INVALID), ((F16, 4096, 8, 1, 32, 4097, 16), ALIGN), ((F32, 4096, 8, 1, 32, 4096, 32), TYPE),
])
def test_round_rows_refusals(gxlib, args, want):
    assert gxlib.lib().gx_quantize_rows(*args, None) == want


@pytest.mark.parametrize("over,want", [
    (dict(type=F32), TYPE), (dict(type_dst=8), TYPE), (dict(rank=0), INVALID), (dict(rank=129), INVALID), (dict(ne00=0), INVALID),
    (dict(ne01=0), INVALID), (dict(n_as=0), INVALID), (dict(n_adapters=0), INVALID), (dict(n_as=4096, n_adapters=3), INVALID),
    (dict(a=None), INVALID), (dict(b=None), INVALID), (dict(x=None), INVALID), (dict(offsets=None), INVALID),
    (dict(base=None), INVALID), (dict(dst=None), INVALID), (dict(ne11=0), INVALID), (dict(n_rows=-1), INVALID),
    (dict(gather=0), INVALID), (dict(nba1=112), INVALID), (dict(nba2=128), INVALID), (dict(nbb1=16), INVALID),
    (dict(nbb2=64), INVALID), (dict(nb11=112), INVALID), (dict(nbb=188), INVALID), (dict(nbd=188), INVALID),
    (dict(nb11=1 << 40), INVALID), (dict(nbb=256, dst=65536), INVALID), (dict(ne01=1 << 30, nbb1=1 << 39, nbb=1 << 33, nbd=1 << 33), INVALID),       # in place with two strides
    (dict(nba1=136), ALIGN), (dict(nbb1=40), ALIGN), (dict(nba2=16 * 128 + 8), ALIGN), (dict(nbb2=48 * 32 + 8), ALIGN),
    (dict(nb11=136), ALIGN), (dict(a=4104), ALIGN), (dict(b=4104), ALIGN), (dict(x=4104), ALIGN), (dict(base=4098), ALIGN),
    (dict(dst=4098), ALIGN), (dict(offsets=4098), ALIGN), (dict(order=4098), ALIGN), (dict(ranks=4098), ALIGN),
    (dict(scale=4098), ALIGN), (dict(nbd=194), ALIGN), (dict(n_rows=0, x=None, base=None, dst=None), OK),
])
def test_lora_refusals(gxlib, over, want):
    import ctypes as C
    a = dict(type=F16, rank=16, ne00=64, ne01=48, n_as=2, n_adapters=4, a=4096, nba1=128, nba2=16 * 128, b=4096, nbb1=32,
             nbb2=48 * 32, ranks=4096, scale=4096)
    c = dict(x=4096, ne11=10, nb11=128, offsets=4096, order=4096, n_rows=10, gather=1, type_dst=F32, base=65536, nbb=192, dst=4096,
             nbd=192)
    assert set(over) <= set(a) | set(c)
    for k, v in over.items():
        (a if k in a else c)[k] = v
    desc = gxlib._lib.gx_lora_desc(*a.values())
    assert gxlib.lib().gx_lora_mul_mat(C.byref(desc), *c.values(), None) == want
    assert gxlib.lib().gx_lora_mul_mat(None, *c.values(), None) == INVALID
