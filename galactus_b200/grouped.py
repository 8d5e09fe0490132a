"""The operators on grouped rows, on torch tensors: rows ordered by expert or
adapter, products with unquantised (F16 / BF16) experts, low-rank adapters of
many requests, rows rounded for them.

Every tensor lives on the current CUDA device. The calls run on `stream` (a
cudaStream_t handle or a torch stream), torch's current stream by default, wait
for nothing and can be captured into a graph. Results they allocate belong to
the stream they run on, as if allocated with it current; what is given (inputs,
`out`, ...) is ordered with it by the caller.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L

_TYPE = {torch.float32: L.TYPE_F32, torch.float16: L.TYPE_F16, torch.bfloat16: L.TYPE_BF16}
_INT = torch.int32
_raw_stream = torch._C._cuda_getCurrentRawStream
_LIB = L.lib()


def _stream(stream, dev: int) -> int:
    if stream is None:
        return _raw_stream(dev)
    return stream if isinstance(stream, int) else int(stream.cuda_stream)


def _new(stream, dev: int, make):
    """What make() allocates, in memory of the stream that the call runs on: a
    block of another stream's could still be read there."""
    if stream is not None:
        handle = stream if isinstance(stream, int) else int(stream.cuda_stream)
        if handle != _raw_stream(dev):
            if isinstance(stream, int):
                stream = torch.cuda.ExternalStream(handle, dev) if handle else torch.cuda.default_stream(dev)
            with torch.cuda.stream(stream):
                return make()
    return make()


def _device(*tensors) -> int:
    """The current device's index; every given tensor must live on it."""
    dev = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"every tensor must be on the current device cuda:{dev}, not {t.device}")
    return dev


def _rows(t, name: str) -> tuple[int, int, int]:
    """(rows, columns, bytes between rows) of a matrix with consecutive elements in its rows."""
    try:
        n, m = t.shape
        s, e = t.stride()
    except ValueError:
        raise ValueError(f"{name}: two dimensions expected, not {tuple(t.shape)}") from None
    if e != 1 and m > 1:
        raise ValueError(f"{name}: consecutive elements in the last dimension expected, not strides {t.stride()}")
    if n <= 1:                                # no second row to reach
        s = (m + 7) & ~7
    return n, m, s * t.element_size()


def _matrices(t, name: str) -> tuple[int, int, int, int, int]:
    """(matrices, rows, columns, bytes between rows, bytes between matrices)."""
    try:
        g, n, m = t.shape
        s0, s1, e = t.stride()
    except ValueError:
        raise ValueError(f"{name}: three dimensions expected, not {tuple(t.shape)}") from None
    if e != 1 and m > 1:
        raise ValueError(f"{name}: consecutive elements in the last dimension expected, not strides {t.stride()}")
    if n <= 1:
        s1 = (m + 7) & ~7
    if g <= 1:
        s0 = n * s1
    size = t.element_size()
    return g, n, m, s1 * size, s0 * size


def _index(t, name: str, n: int | None = None) -> int:
    """Address of an int32 vector (0 for None)."""
    if t is None:
        return 0
    if t.dtype is not _INT or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name}: contiguous int32 vector{'' if n is None else f' of {n}'} expected")
    return t.data_ptr()


def group_rows(ids, n_as: int = 1, *, adapter=None, n_adapters: int = 0, order=None, offsets=None, stream=None):
    """gx_group_rows: ids i32 [T, k] (or None: rows grouped by adapter alone)
    and adapter i32 [T] (or None) -> (order i32 [T*k], offsets i32 [G + 1]),
    G = n_as * max(1, n_adapters). Negative entries take a pair out of every
    group."""
    if ids is not None:
        T, k, nbi1 = _rows(ids, "ids")
        if ids.dtype is not _INT:
            raise ValueError("ids: int32 expected")
        ids_ptr, like = ids.data_ptr(), ids
        adapter_ptr = _index(adapter, "adapter", T)
    elif adapter is not None:
        adapter_ptr, like = _index(adapter, "adapter"), adapter
        T, k, ids_ptr, nbi1 = adapter.shape[0], 1, 0, 0
    else:
        raise ValueError("group_rows: ids or adapter")
    G = n_as * max(1, n_adapters)
    dev = _device(ids, adapter, order, offsets)
    if order is None:
        order = _new(stream, dev, lambda: like.new_empty(T * k))
        order_ptr = order.data_ptr()
    else:
        order_ptr = _index(order, "order", T * k)
    if offsets is None:
        offsets = _new(stream, dev, lambda: like.new_empty(G + 1))
        offsets_ptr = offsets.data_ptr()
    else:
        offsets_ptr = _index(offsets, "offsets", G + 1)
    rc = _LIB.gx_group_rows(ids_ptr, k, T, nbi1, adapter_ptr, n_as, n_adapters, order_ptr, offsets_ptr, _stream(stream, dev))
    if rc:
        L.check(rc, "gx_group_rows")
    return order, offsets


def round_rows(x, dtype, out=None, stream=None):
    """gx_quantize_rows for unquantised weights: f32 rows [rows, n] rounded to float16 or bfloat16."""
    n, m, nb1 = _rows(x, "x")
    if x.dtype != torch.float32 or dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("round_rows: float32 rows to float16 or bfloat16")
    dev = _device(x, out)
    if out is None:
        out = _new(stream, dev, lambda: torch.empty((n, m), dtype=dtype, device=x.device))
    elif out.shape != x.shape or out.dtype != dtype:
        raise ValueError("out: the rows' shape and the given type expected")
    if n and m:
        L.check(_LIB.gx_quantize_rows(_TYPE[dtype], x.data_ptr(), m, n, nb1, out.data_ptr(), _rows(out, "out")[2],
                                      _stream(stream, dev)), "gx_quantize_rows")
    return out


def _product(w, x, offsets, order, n_rows, gather, scatter, out, out_dtype, stream, dev):
    """Common checks and defaults: (result, its type and row stride, the arguments the two products share)."""
    G, N, K, nb01, nb02 = _matrices(w, "weights")
    rows, m, nb11 = _rows(x, "x")
    kind = w.dtype
    if x.dtype is not kind or m != K:
        raise ValueError(f"x: rows of {K} {kind} elements expected, not {m} of {x.dtype}")
    offsets_ptr, order_ptr = _index(offsets, "offsets", G + 1), _index(order, "order")
    if n_rows is None:
        n_rows = rows if order is None else order.shape[0]
    elif order is not None and n_rows > order.shape[0]:
        raise ValueError("n_rows: more than order holds")
    if out is None:
        out = _new(stream, dev, lambda: torch.empty((n_rows, N), dtype=out_dtype or kind, device=w.device))
        nbd1 = N * out.element_size()
    else:
        have, cols, nbd1 = _rows(out, "out")
        if cols != N or have < n_rows or (out_dtype is not None and out.dtype != out_dtype):
            raise ValueError(f"out: at least {n_rows} rows of {N} elements of the result type expected")
    kind_out = _TYPE.get(out.dtype)
    if kind_out is None:
        raise ValueError(f"results of {out.dtype}")
    return out, kind_out, nbd1, (K, N, nb01, nb02, G, x.data_ptr(), rows, nb11, offsets_ptr, order_ptr, n_rows, gather, scatter)


def mul_mat_grouped(w, x, offsets, *, order=None, n_rows: int | None = None, gather: int = 0, scatter: bool = False,
                    out=None, out_dtype=None, stream=None):
    """gx_mul_mat_grouped: weights [G, N, K] and rows [rows, K] of one type
    (float16 or bfloat16), offsets i32 [G + 1] -> [n_rows, N]. Row j of group g
    is x[j], or x[order[j] // gather]; its result goes to row j, or to row
    order[j] with scatter. Rows of no group are left as they were
    (uninitialised in a result allocated here)."""
    dev = _device(w, x, offsets, order, out)
    out, kind, nbd1, args = _product(w, x, offsets, order, n_rows, gather, scatter, out, out_dtype, stream, dev)
    rc = _LIB.gx_mul_mat_grouped(_TYPE.get(w.dtype, -1), w.data_ptr(), *args, kind, out.data_ptr(), nbd1, _stream(stream, dev))
    if rc:
        L.check(rc, "gx_mul_mat_grouped")
    return out


def mul_mat_grouped_glu(gate, up, x, offsets, *, order=None, n_rows: int | None = None, gather: int = 0,
                        scatter: bool = False, act: int = L.ACT_SWIGLU, alpha: float = 1.702, limit: float = 7.0,
                        out=None, out_dtype=None, stream=None):
    """gx_mul_mat_grouped_glu: as mul_mat_grouped with act(gate product, up
    product) in place of the product (ACT_SWIGLU, or ACT_SWIGLU_OAI with alpha
    and limit)."""
    # (strides may differ where no element lies: one expert, one row, one column)
    if up.shape != gate.shape or up.dtype != gate.dtype or \
            up.stride() != gate.stride() and _matrices(up, "up") != _matrices(gate, "gate"):
        raise ValueError("gate and up: one shape, type and layout expected")
    dev = _device(gate, up, x, offsets, order, out)
    out, kind, nbd1, args = _product(gate, x, offsets, order, n_rows, gather, scatter, out, out_dtype, stream, dev)
    rc = _LIB.gx_mul_mat_grouped_glu(_TYPE.get(gate.dtype, -1), gate.data_ptr(), up.data_ptr(), *args, act, alpha, limit, kind,
                                     out.data_ptr(), nbd1, _stream(stream, dev))
    if rc:
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
    G, rank, K, nba1, nba2 = _matrices(a, "a")
    gb, N, rb, nbb1, nbb2 = _matrices(b, "b")
    rows, m, nb11 = _rows(x, "x")
    n_rows, cols, nbb = _rows(base, "base")
    if gb != G or rb != rank or m != K or not a.dtype is b.dtype is x.dtype:
        raise ValueError("a [G, rank, K], b [G, N, rank] and x [rows, K] of one type expected")
    if n_as is None:
        per = ranks if ranks is not None else scale
        n_as = 1 if per is None else G // max(1, per.shape[0])
    if n_as <= 0 or G % n_as:
        raise ValueError("n_as: a divisor of the number of matrices")
    adapters = G // n_as
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != (adapters,) or not scale.is_contiguous()):
        raise ValueError(f"scale: contiguous float32 vector of {adapters} expected")
    dev = _device(a, b, x, offsets, order, ranks, scale, base, out)
    if out is None:
        out = _new(stream, dev, lambda: torch.empty_like(base))
    elif out.shape != base.shape or out.dtype is not base.dtype:
        raise ValueError("out: base's shape and type expected")
    nbd = _rows(out, "out")[2]
    kind = _TYPE.get(base.dtype)
    if cols != N or kind is None:
        raise ValueError(f"base: rows of {N} elements of a result type expected")
    desc = L.gx_lora_desc(_TYPE.get(a.dtype, -1), rank, K, N, n_as, adapters, a.data_ptr(), nba1, nba2, b.data_ptr(), nbb1, nbb2,
                          _index(ranks, "ranks", adapters), 0 if scale is None else scale.data_ptr())
    rc = _LIB.gx_lora_mul_mat(C.byref(desc), x.data_ptr(), rows, nb11, _index(offsets, "offsets", G + 1),
                              _index(order, "order", n_rows), n_rows, gather, kind, base.data_ptr(), nbb, out.data_ptr(), nbd,
                              _stream(stream, dev))
    if rc:
        L.check(rc, "gx_lora_mul_mat")
    return out
