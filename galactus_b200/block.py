"""Products with 4-bit weights and the norms around a block, on torch tensors.

Every tensor lives on the current CUDA device; streams, captures and the memory
of results are as in the operators on grouped rows.
"""
from __future__ import annotations

import struct

import torch

from . import _lib as L
from .grouped import _INT, _TYPE, _device, _index, _matrices, _new, _rows, _stream

_LIB = L.lib()
_F32 = torch.float32
_CALLS = {"gx_mul_mat_q4": _LIB.gx_mul_mat_q4, "gx_mul_mat_q4_glu": _LIB.gx_mul_mat_q4_glu}


def _q4(name, w, up, x, type, ids, offsets, order, n_rows, gather, scatter, act, out, out_dtype, stream):
    dev = _device(w, up, x, ids, offsets, order, out)
    G, N, nb, nb01, nb02 = _matrices(w, "weights")
    if w.dtype is not torch.uint8:
        raise ValueError(f"weights: uint8 rows of blocks expected, not {w.dtype}")
    if w.shape[1] <= 1:                      # (one row: no second one to reach)
        nb01 = (nb + 3) & ~3
    if G <= 1:
        nb02 = N * nb01
    rows, K, nb11 = _rows(x, "x")
    if type not in (L.TYPE_Q4_0, L.TYPE_Q4_1) or K % 64 or L.row_bytes(type, K) != nb:
        raise ValueError(f"weights: rows of {K} elements (a multiple of 64) in blocks of TYPE_Q4_0 or TYPE_Q4_1 expected")
    if ids is not None:
        if offsets is not None or order is not None:
            raise ValueError("ids, or offsets and order")
        if ids.dtype is not _INT or not ids.is_contiguous():
            raise ValueError("ids: contiguous int32 expected")
        if n_rows is None:
            n_rows = ids.numel()
        elif n_rows > ids.numel():
            raise ValueError("n_rows: more than ids holds")
        ids_ptr, offsets_ptr, order_ptr = ids.data_ptr(), 0, 0
    else:
        ids_ptr, offsets_ptr, order_ptr = 0, _index(offsets, "offsets", G + 1), _index(order, "order")
        if n_rows is None:
            n_rows = rows if order is None else order.shape[0]
        elif order is not None and n_rows > order.shape[0]:
            raise ValueError("n_rows: more than order holds")
    if out is None:
        kind = out_dtype or x.dtype
        out = x.new_empty((n_rows, N), dtype=kind) if stream is None else _new(stream, dev, lambda: x.new_empty((n_rows, N), dtype=kind))
        nbd1 = N * out.element_size()
    else:
        have, cols, nbd1 = _rows(out, "out")
        if cols != N or have < n_rows or (out_dtype is not None and out.dtype != out_dtype):
            raise ValueError(f"out: at least {n_rows} rows of {N} elements of the result type expected")
    kind = _TYPE.get(out.dtype)
    if kind is None:
        raise ValueError(f"results of {out.dtype}")
    b_type = _TYPE.get(x.dtype, -1)
    head = (type, w.data_ptr()) if up is None else (type, w.data_ptr(), up.data_ptr())
    rc = _CALLS[name](*head, K, N, nb01, nb02, G, b_type, x.data_ptr(), rows, nb11, ids_ptr, offsets_ptr, order_ptr, n_rows,
                             gather, scatter, *act, kind, out.data_ptr(), nbd1, _stream(stream, dev))
    if rc:
        L.check(rc, name)
    return out


def mul_mat_q4(w, x, *, type: int, ids=None, offsets=None, order=None, n_rows: int | None = None, gather: int = 0,
               scatter: bool = False, out=None, out_dtype=None, stream=None):
    """gx_mul_mat_q4: weights uint8 [G, N, bytes] (rows of TYPE_Q4_0 or
    TYPE_Q4_1 blocks), rows x [rows, K] of float16 or bfloat16 -> [n_rows, N].

    ids (int32, any contiguous shape, at most 256 of them): row j = x[j //
    gather] times the matrix ids[j], to result row j; rows of negative ids are
    left as they were (uninitialised in a result allocated here); many rows of
    one matrix are faster as a group. offsets (and order): the groups of
    group_rows, as in mul_mat_grouped. Neither: one matrix for all rows."""
    return _q4("gx_mul_mat_q4", w, None, x, type, ids, offsets, order, n_rows, gather, scatter, (), out, out_dtype, stream)


def mul_mat_q4_glu(gate, up, x, *, type: int, ids=None, offsets=None, order=None, n_rows: int | None = None, gather: int = 0,
                   scatter: bool = False, act: int = L.ACT_SWIGLU, alpha: float = 1.702, limit: float = 7.0, out=None,
                   out_dtype=None, stream=None):
    """gx_mul_mat_q4_glu: as mul_mat_q4 with act(gate product, up product) in
    place of the product (ACT_SWIGLU, or ACT_SWIGLU_OAI with alpha and limit)."""
    if up.shape != gate.shape or up.dtype != gate.dtype or \
            up.stride() != gate.stride() and _matrices(up, "up") != _matrices(gate, "gate"):
        raise ValueError("gate and up: one shape, type and layout expected")
    return _q4("gx_mul_mat_q4_glu", gate, up, x, type, ids, offsets, order, n_rows, gather, scatter, (act, alpha, limit), out,
               out_dtype, stream)


# gx_block_desc, field by field (a structure's attributes, set one by one, took 5 us)
_DESC = struct.Struct("@2q6i P2q2P P q 2P 2f P2q i f P q P q P q P")
assert _DESC.size == L.C.sizeof(L.gx_block_desc)


def _result(t, like, rows, cols, dtype, name, stream, dev):
    """(tensor, its type, bytes between its rows): t, or a new one."""
    if t is None:
        if stream is None:
            t = like.new_empty((rows, cols), dtype=dtype)
        else:
            t = _new(stream, dev, lambda: like.new_empty((rows, cols), dtype=dtype))
        kind = _TYPE.get(dtype)
        if kind is None:
            raise ValueError(f"{name}: results of {dtype}")
        return t, kind, cols * t.element_size()
    if tuple(t.shape) != (rows, cols) or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{name}: {(rows, cols)} of the result type expected")
    kind = _TYPE.get(t.dtype)
    if kind is None:
        raise ValueError(f"{name}: results of {t.dtype}")
    return t, kind, _rows(t, name)[2]


def _vector(t, name, n):
    if t is None:
        return 0
    if t.dtype is not _F32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous float32 vector of {n} expected")
    return t.data_ptr()


def _given(t, name, rows, cols):
    """(type, address, bytes between rows) of rows that may be absent."""
    if t is None:
        return 0, 0, 0
    n, m, nb = _rows(t, name)
    if n != rows or m != cols:
        raise ValueError(f"{name}: [{rows}, {cols}] expected")
    return _TYPE.get(t.dtype, -1), t.data_ptr(), nb


def rms_norm(x, weight=None, *, eps: float = 1e-6, out=None, out_dtype=None, stream=None):
    """gx_rms_norm: rows x [T, H] / sqrt(mean(x^2) + eps) * weight (float32 [H], or ones)."""
    T, H, nb1 = _rows(x, "x")
    dev = _device(x, weight, out)
    out, kind, nbd = _result(out, x, T, H, out_dtype or (x.dtype if out is None else None), "out", stream, dev)
    rc = _LIB.gx_rms_norm(_TYPE.get(x.dtype, -1), x.data_ptr(), H, T, nb1, _vector(weight, "weight", H), eps, kind, out.data_ptr(), nbd,
                          _stream(stream, dev))
    if rc:
        L.check(rc, "gx_rms_norm")
    return out


def block_out(y, *, weights=None, ids=None, shared=None, shared_gate=None, norm=None, eps: float = 1e-6, gate=None,
              gate_sigmoid: bool = False, scale: float = 1.0, residual=None, out=None, out_dtype=None, next_norm=None,
              next_dtype=None, next_out=None, next_eps: float | None = None, stream=None):
    """gx_block_out: the end of a block. y [T, k, H] (or [T, H]), weights
    float32 and ids int32 [T, k], shared [T, H] with shared_gate float32 [T],
    norm float32 [H], gate float32 [T or 1, H or 1], residual [T, H] ->
    out [T, H] (of the residual's type, y's without one), and with next_norm
    (float32 [H]), next_dtype or next_out the pair (out, the next block's normed
    rows)."""
    shape, strides = y.shape, y.stride()
    if len(shape) == 2:
        shape, strides = (shape[0], 1, shape[1]), (strides[0], 0, strides[1])
    if len(shape) != 3 or (shape[2] > 1 and strides[2] != 1):
        raise ValueError("y: [T, k, H] with consecutive elements in its rows expected")
    T, k, H = shape
    dev = _device(y, weights, ids, shared, shared_gate, norm, gate, residual, out, next_norm, next_out)
    size = y.element_size()
    ids_ptr = 0
    if ids is not None:
        if ids.dtype is not _INT or ids.numel() != T * k or not ids.is_contiguous():
            raise ValueError(f"ids: contiguous int32 [{T}, {k}] expected")
        ids_ptr = ids.data_ptr()
    type_shared, shared_ptr, nbs = _given(shared, "shared", T, H)
    type_residual, residual_ptr, nbr = _given(residual, "residual", T, H)
    gate_ptr = gne0 = nbg = 0
    if gate is not None:
        rows, gne0, nbg = _rows(gate, "gate")
        if gate.dtype is not _F32 or rows not in (1, T) or gne0 not in (1, H):
            raise ValueError(f"gate: float32 [{T} or 1, {H} or 1] expected")
        gate_ptr = gate.data_ptr()
        if rows == 1:
            nbg = 0
    if out_dtype is None and out is None:
        out_dtype = y.dtype if residual is None else residual.dtype
    out, type_dst, nbd = _result(out, y, T, H, out_dtype, "out", stream, dev)
    more = next_norm is not None or next_dtype is not None or next_out is not None
    type_next = next_ptr = nbn = 0
    if more:
        next_out, type_next, nbn = _result(next_out, y, T, H, next_dtype or (y.dtype if next_out is None else None), "next_out", stream,
                                           dev)
        next_ptr = next_out.data_ptr()
    desc = _DESC.pack(H, T, k, _TYPE.get(y.dtype, -1), type_shared, type_residual, type_dst, type_next, y.data_ptr(),
                      (strides[1] if k > 1 else H) * size, (strides[0] if T > 1 else k * H) * size, _vector(weights, "weights", T * k),
                      ids_ptr, shared_ptr, nbs, _vector(shared_gate, "shared_gate", T), _vector(norm, "norm", H), eps, scale, gate_ptr,
                      gne0, nbg, L.GATE_SIGMOID if gate_sigmoid else L.GATE_NONE, eps if next_eps is None else next_eps, residual_ptr,
                      nbr, out.data_ptr(), nbd, next_ptr, nbn, _vector(next_norm, "next_norm", H))
    rc = _LIB.gx_block_out(desc, _stream(stream, dev))
    if rc:
        L.check(rc, "gx_block_out")
    return (out, next_out) if more else out
