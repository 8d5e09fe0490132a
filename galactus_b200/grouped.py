"""The operators on grouped rows, on torch tensors: rows ordered by expert or
adapter, products with unquantised (F16 / BF16) experts, low-rank adapters of
many requests, rows rounded for them.

Every tensor lives on the current CUDA device. The calls run on `stream` (a
cudaStream_t handle or a torch stream), torch's current stream by default, wait
for nothing and can be captured into a graph; results they allocate belong to
torch's current stream.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L

_TYPE = {torch.float32: L.TYPE_F32, torch.float16: L.TYPE_F16, torch.bfloat16: L.TYPE_BF16}


def _raw_stream(stream, dev: int) -> int:
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(dev)
    return stream if isinstance(stream, int) else int(stream.cuda_stream)


def _device(*tensors) -> int:
    """The current device's index; every given tensor must live on it."""
    dev = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"every tensor must be on the current device cuda:{dev}, not {t.device}")
    return dev


def _matrix(t, name: str, dims: int) -> None:
    if t.dim() != dims or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name}: {dims} dimensions with consecutive elements in the last one, not shape {tuple(t.shape)} "
                         f"strides {t.stride()}")


def _index(t, name: str, n: int | None = None) -> None:
    if t is None:
        return
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name}: contiguous int32 vector{'' if n is None else f' of {n}'} expected")


def _row_stride(t, dim: int) -> int:
    """Bytes between consecutive entries of a dimension; of no consequence, and so the packed value, where there is one."""
    if t.shape[dim] > 1:
        return t.stride(dim) * t.element_size()
    n = t.element_size()
    for s in t.shape[dim + 1:]:
        n *= s
    return (n + 15) // 16 * 16


def group_rows(ids, n_as: int = 1, *, adapter=None, n_adapters: int = 0, order=None, offsets=None, stream=None):
    """gx_group_rows: ids i32 [T, k] (or None: rows grouped by adapter alone)
    and adapter i32 [T] (or None) -> (order i32 [T*k], offsets i32 [G + 1]),
    G = n_as * max(1, n_adapters). Negative entries take a pair out of every
    group."""
    if ids is None and adapter is None:
        raise ValueError("group_rows: ids or adapter")
    dev = _device(ids, adapter, order, offsets)
    _index(adapter, "adapter", None if ids is None else ids.shape[0])
    if ids is not None:
        _matrix(ids, "ids", 2)
        if ids.dtype != torch.int32:
            raise ValueError("ids: int32 expected")
        T, k = ids.shape
        ids_ptr, nbi1 = ids.data_ptr(), _row_stride(ids, 0) if T > 1 else 4 * k
    else:
        T, k, ids_ptr, nbi1 = adapter.shape[0], 1, 0, 0
    G = n_as * max(1, n_adapters)
    where = adapter.device if ids is None else ids.device
    if order is None:
        order = torch.empty(T * k, dtype=torch.int32, device=where)
    if offsets is None:
        offsets = torch.empty(G + 1, dtype=torch.int32, device=where)
    _index(order, "order", T * k)
    _index(offsets, "offsets", G + 1)
    rc = L.lib().gx_group_rows(ids_ptr, k, T, nbi1, 0 if adapter is None else adapter.data_ptr(), n_as, n_adapters,
                               order.data_ptr(), offsets.data_ptr(), _raw_stream(stream, dev))
    L.check(rc, "gx_group_rows")
    return order, offsets


def round_rows(x, dtype, out=None, stream=None):
    """gx_quantize_rows for unquantised weights: f32 rows [rows, n] rounded to float16 or bfloat16."""
    dev = _device(x, out)
    _matrix(x, "x", 2)
    if x.dtype != torch.float32 or dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("round_rows: float32 rows to float16 or bfloat16")
    if out is None:
        out = torch.empty(x.shape, dtype=dtype, device=x.device)
    _matrix(out, "out", 2)
    if out.shape != x.shape or out.dtype != dtype:
        raise ValueError("out: the rows' shape and the given type expected")
    if x.numel():
        L.check(L.lib().gx_quantize_rows(_TYPE[dtype], x.data_ptr(), x.shape[1], x.shape[0], _row_stride(x, 0),
                                         out.data_ptr(), _row_stride(out, 0), _raw_stream(stream, dev)),
                "gx_quantize_rows")
    return out


def _product(w, x, offsets, order, n_rows, gather, scatter, out, out_dtype):
    """Common checks and defaults; the arguments the two products share."""
    _matrix(w, "weights", 3)
    _matrix(x, "x", 2)
    if x.dtype != w.dtype or x.shape[1] != w.shape[2]:
        raise ValueError(f"x: rows of {w.shape[2]} {w.dtype} elements expected, not {x.shape[1]} of {x.dtype}")
    _index(offsets, "offsets", w.shape[0] + 1)
    _index(order, "order")
    if n_rows is None:
        n_rows = x.shape[0] if order is None else order.shape[0]
    elif order is not None and n_rows > order.shape[0]:
        raise ValueError("n_rows: more than order holds")
    if out is None:
        out = torch.empty((n_rows, w.shape[1]), dtype=out_dtype or w.dtype, device=w.device)
    else:
        _matrix(out, "out", 2)
        if out.shape[1] != w.shape[1] or out.shape[0] < n_rows or (out_dtype is not None and out.dtype != out_dtype):
            raise ValueError(f"out: at least {n_rows} rows of {w.shape[1]} elements of the result type expected")
    if out.dtype not in _TYPE:
        raise ValueError(f"results of {out.dtype}")
    tail = (w.shape[2], w.shape[1], _row_stride(w, 1), _row_stride(w, 0), w.shape[0], x.data_ptr(), x.shape[0],
            _row_stride(x, 0), offsets.data_ptr(), 0 if order is None else order.data_ptr(), n_rows, gather, int(scatter))
    return out, tail


def mul_mat_grouped(w, x, offsets, *, order=None, n_rows: int | None = None, gather: int = 0, scatter: bool = False,
                    out=None, out_dtype=None, stream=None):
    """gx_mul_mat_grouped: weights [G, N, K] and rows [rows, K] of one type
    (float16 or bfloat16), offsets i32 [G + 1] -> [n_rows, N]. Row j of group g
    is x[j], or x[order[j] // gather]; its result goes to row j, or to row
    order[j] with scatter. Rows of no group are left as they were
    (uninitialised in a result allocated here)."""
    dev = _device(w, x, offsets, order, out)
    out, tail = _product(w, x, offsets, order, n_rows, gather, scatter, out, out_dtype)
    rc = L.lib().gx_mul_mat_grouped(_TYPE.get(w.dtype, -1), w.data_ptr(), *tail, _TYPE[out.dtype], out.data_ptr(),
                                    _row_stride(out, 0), _raw_stream(stream, dev))
    L.check(rc, "gx_mul_mat_grouped")
    return out


def mul_mat_grouped_glu(gate, up, x, offsets, *, order=None, n_rows: int | None = None, gather: int = 0,
                        scatter: bool = False, act: int = L.ACT_SWIGLU, alpha: float = 1.702, limit: float = 7.0,
                        out=None, out_dtype=None, stream=None):
    """gx_mul_mat_grouped_glu: as mul_mat_grouped with act(gate product, up
    product) in place of the product (ACT_SWIGLU, or ACT_SWIGLU_OAI with alpha
    and limit)."""
    dev = _device(gate, up, x, offsets, order, out)
    _matrix(up, "up", 3)
    if up.shape != gate.shape or up.dtype != gate.dtype or \
            (_row_stride(up, 0), _row_stride(up, 1)) != (_row_stride(gate, 0), _row_stride(gate, 1)):
        raise ValueError("gate and up: one shape, type and layout expected")
    out, tail = _product(gate, x, offsets, order, n_rows, gather, scatter, out, out_dtype)
    rc = L.lib().gx_mul_mat_grouped_glu(_TYPE.get(gate.dtype, -1), gate.data_ptr(), up.data_ptr(), *tail, act, alpha, limit,
                                        _TYPE[out.dtype], out.data_ptr(), _row_stride(out, 0), _raw_stream(stream, dev))
    L.check(rc, "gx_mul_mat_grouped_glu")
    return out


def lora_mul_mat(a, b, x, offsets, *, order=None, gather: int = 1, n_as: int | None = None, ranks=None, scale=None, base,
                 out=None, stream=None):
    """gx_lora_mul_mat: base + the rows' low-rank deltas, in a new tensor, in
    `out`, or in place (out=base). a [G, rank, K] and b [G, N, rank] hold the
    adapters (G = adapters * n_as, expert minor), x [rows, K] the projection's
    input of their type, base [n_rows, N] its output; ranks i32 and scale f32
    [adapters] (n_as defaults to G // len(ranks or scale), else 1). order and
    offsets as group_rows gives them; row r of base belongs to x[r // gather]."""
    dev = _device(a, b, x, offsets, order, ranks, scale, base, out)
    for t, name, dims in ((a, "a", 3), (b, "b", 3), (x, "x", 2), (base, "base", 2)):
        _matrix(t, name, dims)
    G, rank, K = a.shape
    if b.shape[0] != G or b.shape[2] != rank or not a.dtype == b.dtype == x.dtype or x.shape[1] != K:
        raise ValueError("a [G, rank, K], b [G, N, rank] and x [rows, K] of one type expected")
    if n_as is None:
        per = ranks if ranks is not None else scale
        n_as = 1 if per is None else G // max(1, per.shape[0])
    if n_as <= 0 or G % n_as:
        raise ValueError("n_as: a divisor of the number of matrices")
    adapters = G // n_as
    _index(offsets, "offsets", G + 1)
    _index(order, "order", base.shape[0])
    _index(ranks, "ranks", adapters)
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != (adapters,) or not scale.is_contiguous()):
        raise ValueError(f"scale: contiguous float32 vector of {adapters} expected")
    if out is None:
        out = torch.empty(base.shape, dtype=base.dtype, device=base.device)
    _matrix(out, "out", 2)
    if base.shape[1] != b.shape[1] or out.shape != base.shape or out.dtype != base.dtype or base.dtype not in _TYPE:
        raise ValueError(f"base and out: rows of {b.shape[1]} elements of one result type expected")
    desc = L.gx_lora_desc(_TYPE.get(a.dtype, -1), rank, K, b.shape[1], n_as, adapters, a.data_ptr(), _row_stride(a, 1),
                          _row_stride(a, 0), b.data_ptr(), _row_stride(b, 1), _row_stride(b, 0),
                          None if ranks is None else ranks.data_ptr(), None if scale is None else scale.data_ptr())
    rc = L.lib().gx_lora_mul_mat(C.byref(desc), x.data_ptr(), x.shape[0], _row_stride(x, 0), offsets.data_ptr(),
                                 0 if order is None else order.data_ptr(), base.shape[0], gather, _TYPE[base.dtype],
                                 base.data_ptr(), _row_stride(base, 0), out.data_ptr(), _row_stride(out, 0),
                                 _raw_stream(stream, dev))
    L.check(rc, "gx_lora_mul_mat")
    return out
