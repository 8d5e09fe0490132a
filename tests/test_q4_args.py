"""Host-side checks of the products with 4-bit weights and of the norms around
a block: every refusal happens before any device work, so it is the same with
and without a GPU."""
import ctypes as C

import pytest

F32, F16, BF16, Q4_0, Q4_1 = 0, 1, 30, 2, 3
OK, INVALID, TYPE, ALIGN = 0, -1, -2, -3
PRODUCT = dict(type=Q4_0, w=4096, ne00=64, ne01=48, nb01=36, nb02=48 * 36, n_as=4, type_b=BF16, b=4096, ne11=10, nb11=128, ids=None,
               offsets=4096, order=4096, n_rows=10, gather=0, scatter=0, type_dst=F32, dst=4096, nbd1=192)
NO_GROUPS = dict(offsets=None, order=None)


def product(gxlib, **over):
    assert set(over) <= set(PRODUCT)
    return gxlib.lib().gx_mul_mat_q4(*{**PRODUCT, **over}.values(), None)


def glu(gxlib, **over):
    a = {}
    for k, v in PRODUCT.items():
        a["gate" if k == "w" else k] = v
        if k == "w":
            a["up"] = 8192
        if k == "scatter":
            a.update(act=0, alpha=1.702, limit=7.0)
    assert set(over) <= set(a)
    return gxlib.lib().gx_mul_mat_q4_glu(*{**a, **over}.values(), None)


COMMON = [
    (dict(type=F16), TYPE), (dict(type=8), TYPE), (dict(type=39), TYPE), (dict(type_b=F32), TYPE), (dict(type_dst=Q4_0), TYPE),
    (dict(ne00=0), INVALID), (dict(ne01=0), INVALID), (dict(n_as=0), INVALID), (dict(n_as=8193), INVALID), (dict(n_rows=-1), INVALID),
    (dict(gather=-1), INVALID), (dict(scatter=2), INVALID), (dict(nb01=32), INVALID), (dict(nb02=47 * 36), INVALID),
    (dict(type=Q4_1), INVALID), (dict(nb11=112), INVALID), (dict(nbd1=188), INVALID), (dict(nb01=1 << 40), INVALID),
    (dict(ne11=9), INVALID), (dict(ne11=0), INVALID), (dict(b=None), INVALID), (dict(dst=None), INVALID),
    (dict(order=None, scatter=1), INVALID), (dict(order=None, gather=2), INVALID),
    (dict(offsets=None), INVALID), (dict(**NO_GROUPS), INVALID),                       # four matrices, none named
    (dict(ids=4096), INVALID), (dict(ids=4096, offsets=None), INVALID), (dict(ids=4096, order=None), INVALID),
    (dict(ids=4096, n_rows=257, ne11=257, **NO_GROUPS), INVALID), (dict(ids=4096, ne11=9, gather=1, **NO_GROUPS), INVALID),
    (dict(ids=4096, ne11=9, **NO_GROUPS), INVALID),
    (dict(ne00=96, nb01=54, nb02=48 * 54, nb11=192), ALIGN), (dict(nb01=38, nb02=48 * 38), ALIGN), (dict(nb02=48 * 36 + 2), ALIGN),
    (dict(nb11=136), ALIGN), (dict(b=4104), ALIGN), (dict(offsets=4098), ALIGN), (dict(order=4097), ALIGN), (dict(dst=4098), ALIGN),
    (dict(ids=4098, **NO_GROUPS), ALIGN), (dict(nbd1=194), ALIGN),
    (dict(n_rows=0, b=None, dst=None, order=None, offsets=None, ne11=0), OK),
    (dict(ne01=1 << 30, nb01=1 << 39, nb02=1 << 39, nbd1=1 << 33), INVALID),          # a matrix of 2^69 bytes
]


@pytest.mark.parametrize("over,want", COMMON + [(dict(w=None), INVALID), (dict(w=4104), ALIGN)])
def test_product_refusals(gxlib, over, want):
    assert product(gxlib, **over) == want


@pytest.mark.parametrize("over,want", COMMON + [(dict(gate=None), INVALID), (dict(up=None), INVALID), (dict(up=8200), ALIGN),
                                                (dict(gate=4104), ALIGN), (dict(act=2), INVALID)])
def test_glu_refusals(gxlib, over, want):
    assert glu(gxlib, **over) == want


@pytest.mark.parametrize("over,want", [
    (dict(type_src=Q4_0), TYPE), (dict(type_dst=8), TYPE), (dict(ne0=0), INVALID), (dict(ne0=65537), INVALID), (dict(ne1=-1), INVALID),
    (dict(nb1=252), INVALID), (dict(nbd1=126), INVALID), (dict(nb1=258), ALIGN), (dict(nbd1=129), ALIGN), (dict(src=None), INVALID),
    (dict(dst=None), INVALID), (dict(src=4098), ALIGN), (dict(dst=4097), ALIGN), (dict(weight=4098), ALIGN), (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(nb1=1 << 40), INVALID), (dict(ne1=1 << 31), INVALID),
    (dict(ne1=0, src=None, dst=None), OK),
])
def test_norm_refusals(gxlib, over, want):
    a = dict(type_src=F32, src=4096, ne0=64, ne1=3, nb1=256, weight=4096, eps=1e-6, type_dst=F16, dst=4096, nbd1=128)
    assert set(over) <= set(a)
    a.update(over)
    assert gxlib.lib().gx_rms_norm(*a.values(), None) == want


@pytest.mark.parametrize("over,want", [
    (dict(ne0=0), INVALID), (dict(ne0=65537), INVALID), (dict(ne1=-1), INVALID), (dict(k=0), INVALID), (dict(ne1=1 << 20, k=1 << 14), INVALID),
    (dict(y=None), INVALID), (dict(dst=None, next=None), INVALID), (dict(shared=None), INVALID), (dict(eps=-1.0), INVALID),
    (dict(next_eps=-1.0), INVALID), (dict(type_y=Q4_0), TYPE), (dict(type_shared=8), TYPE), (dict(type_residual=8), TYPE),
    (dict(type_dst=8), TYPE), (dict(type_next=8), TYPE), (dict(nby1=252), INVALID), (dict(nby2=252), INVALID), (dict(nbs=126), INVALID),
    (dict(nbr=252), INVALID), (dict(nbd=252), INVALID), (dict(nbn=126), INVALID), (dict(nby1=258), ALIGN), (dict(y=4098), ALIGN),
    (dict(shared=4097), ALIGN), (dict(residual=4098), ALIGN), (dict(dst=4098), ALIGN), (dict(next=4097), ALIGN), (dict(weights=4098), ALIGN),
    (dict(ids=4098), ALIGN), (dict(shared_gate=4098), ALIGN), (dict(norm=4098), ALIGN), (dict(next_norm=4098), ALIGN),
    (dict(gate=4098), ALIGN), (dict(gne0=2), INVALID), (dict(nbg=128), INVALID), (dict(nbg=258), ALIGN), (dict(gate_act=2), INVALID),
    (dict(ne1=0, y=None, dst=None, next=None), OK),
])
def test_block_refusals(gxlib, over, want):
    a = dict(ne0=64, ne1=3, k=2, type_y=F32, type_shared=F16, type_residual=F32, type_dst=F32, type_next=BF16, y=4096, nby1=256, nby2=512,
             weights=4096, ids=4096, shared=4096, nbs=128, shared_gate=4096, norm=4096, eps=1e-6, scale=1.0, gate=4096, gne0=64, nbg=256,
             gate_act=0, next_eps=1e-6, residual=4096, nbr=256, dst=8192, nbd=256, next=16384, nbn=128, next_norm=4096)
    assert set(over) <= set(a) and [n for n, _ in gxlib._lib.gx_block_desc._fields_] == list(a)
    a.update(over)
    desc = gxlib._lib.gx_block_desc(*a.values())
    assert gxlib.lib().gx_block_out(C.byref(desc), None) == want
    assert gxlib.lib().gx_block_out(None, None) == INVALID
