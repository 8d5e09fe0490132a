"""Sizes whose tiles 32 bits would not count are refused on the host."""
import ctypes as C

import pytest

F32, BF16, INVALID = 0, 30, -1
BIG = (1 << 31) - 1
LIMIT = BIG - 65536


@pytest.mark.parametrize("size", [BIG, LIMIT + 1])
@pytest.mark.parametrize("over", ["ne00", "ne01", "ne11", "n_rows"])
def test_products(gxlib, over, size):
    a = dict(type=BF16, w=4096, ne00=64, ne01=48, nb01=1 << 33, nb02=1 << 39, n_as=1, b=4096, ne11=BIG if over == "n_rows" else 10,
             nb11=1 << 33, offsets=4096, order=4096, n_rows=10, gather=0, scatter=0, type_dst=F32, dst=4096, nbd1=1 << 35)
    a[over] = size
    assert gxlib.lib().gx_mul_mat_grouped(*a.values(), None) == INVALID
    g = dict(type=a.pop("type"), gate=a.pop("w"), up=4096, **a)
    tail = [g.pop(n) for n in ("type_dst", "dst", "nbd1")]
    assert gxlib.lib().gx_mul_mat_grouped_glu(*g.values(), 0, 1.0, 7.0, *tail, None) == INVALID


@pytest.mark.parametrize("size", [BIG, LIMIT + 1])
@pytest.mark.parametrize("over", ["ne00", "ne01", "ne11", "n_rows"])
def test_adapters(gxlib, over, size):
    a = dict(type=BF16, rank=16, ne00=64, ne01=48, n_as=1, n_adapters=1, a=4096, nba1=1 << 33, nba2=1 << 39, b=4096, nbb1=1 << 6,
             nbb2=1 << 39, ranks=4096, scale=4096)
    c = dict(x=4096, ne11=10, nb11=1 << 33, offsets=4096, order=4096, n_rows=10, gather=1, type_dst=F32, base=65536, nbb=1 << 35,
             dst=4096, nbd=1 << 35)
    (a if over in a else c)[over] = size
    desc = gxlib._lib.gx_lora_desc(*a.values())
    assert gxlib.lib().gx_lora_mul_mat(C.byref(desc), *c.values(), None) == INVALID
