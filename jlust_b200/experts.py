"""A layer of experts: the routing pattern, the products grouped by expert and
the dense product with its epilogue, with their gradients.

A token's k expert indices are one row of a sparse tokens x experts matrix.
`route` compresses its pattern by expert on the GPU without a host
synchronisation; `grouped_matmul` is the product with the block-diagonal matrix
of the experts' weights, whose blocks have ragged row ranges; `combine` adds a
token's rows back together with its weights.  `fused_matmul` is the product of
one group: act(x W + b) + r.  No counterpart in the reference.

Values are BF16 or F32, one type for a call's operands, with fp32 sums.
Gradients are deterministic: no atomics.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .backend import AbstractKernelHandle
from .errors import (DeviceMismatch, IncompatibleExtents, InvalidArgument,
                     UnsupportedIndexType, UnsupportedValueType)
from .tensor import _origin

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_ACTS = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "relu": _lib.ACT_RELU,
         "silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}


# The calls below are short on the GPU, so their host side is kept lean:
# addresses go to ctypes as integers and each operand is looked at once.

def _base(origin) -> int:
    return 0 if origin == 0 else _origin(origin).offset


def _on(t: torch.Tensor) -> torch.device:
    """The CUDA device of a call's first operand."""
    d = t.device
    if d.type != "cuda":
        raise DeviceMismatch(f"B200Backend runs on CUDA devices only (operands on {d}); "
                             "there is no CPU fallback")
    return d


# The current stream's handle without building a Stream object (2 us a call)
# where this torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _act(act) -> int:
    try:
        return _ACTS[act]
    except (KeyError, TypeError):
        raise InvalidArgument(f"unknown activation {act!r} (none, relu, silu, gelu)") from None


def _type(t: torch.Tensor, what: str) -> int:
    try:
        return _TYPES[t.dtype]
    except KeyError:
        raise UnsupportedValueType(f"{what}: value type {t.dtype} (Float32 or BFloat16)") from None


def _rows(t: torch.Tensor, rows, cols, what: str, like: torch.Tensor):
    """Leading dimension of a row-major rows x cols matrix of like's type."""
    if t.dim() != 2 or t.shape != (rows, cols):
        raise IncompatibleExtents(f"{what} is {tuple(t.shape)}, expected ({rows}, {cols})")
    if t.dtype != like.dtype:
        raise UnsupportedValueType(f"{what}: operands must share one value type "
                                   f"({t.dtype}, {like.dtype})")
    if t.device != like.device:
        raise _elsewhere(t, like, what)
    s0, s1 = t.stride()
    if cols > 1 and s1 != 1 or rows > 1 and s0 < cols:
        raise IncompatibleExtents(f"{what} must be row-major (strides {t.stride()})")
    return s0 if rows > 1 and s0 > 0 else max(cols, 1)


def _elsewhere(t, like, what):
    return DeviceMismatch(f"{what} lives on {t.device}, the other operands on {like.device}")


def _index(t: torch.Tensor, n, what: str, like: torch.Tensor):
    if t.dtype != torch.int32:
        raise UnsupportedIndexType(f"{what}: index buffers must be Int32 (got {t.dtype})")
    if t.numel() != n or not t.is_contiguous():
        raise IncompatibleExtents(f"{what} must be {n} contiguous indices (has {t.numel()})")
    if t.device != like.device:
        raise _elsewhere(t, like, what)


def _matrix(K, N, s0, s1, strides):
    """(leading dimension, order) of a K x N matrix of strides s0, s1."""
    if (s1 == 1 or N <= 1) and (s0 >= N or K <= 1):
        return (s0 if K > 1 else max(N, 1)), _lib.ROW_MAJOR
    if (s0 == 1 or K <= 1) and (s1 >= K or N <= 1):
        return (s1 if N > 1 else max(K, 1)), _lib.COL_MAJOR
    raise IncompatibleExtents(f"w's matrices must be row- or column-major (strides {strides})")


def _weight(w: torch.Tensor):
    """(E, K, N, leading dimension, expert stride, order) of E x K x N weights,
    or of one K x N matrix, row- or column-major."""
    strides = w.stride()
    if w.dim() == 3:
        E, K, N = w.shape
        ld, order = _matrix(K, N, strides[1], strides[2], strides)
        if E > 1:
            return E, K, N, ld, strides[0], order
    elif w.dim() == 2:
        E, (K, N) = 1, w.shape
        ld, order = _matrix(K, N, strides[0], strides[1], strides)
    else:
        raise IncompatibleExtents(f"w must be experts x K x N or K x N (got {tuple(w.shape)})")
    return E, K, N, ld, ld * (K if order == _lib.ROW_MAJOR else N), order


def _experts(w):
    if w.dim() != 3:
        raise IncompatibleExtents(f"w must be experts x K x N (got {tuple(w.shape)})")
    return w


def _dense(w):
    if w.dim() != 2:
        raise IncompatibleExtents(f"w must be K x N (got {tuple(w.shape)})")
    return w


def _bias(bias, E, N, w):
    if bias is None:
        return 0
    if bias.dim() == 2:
        return _rows(bias, E, N, "bias", w)
    if E != 1 or bias.shape != (N,) or (N > 1 and bias.stride(0) != 1):
        raise IncompatibleExtents(f"bias is {tuple(bias.shape)}, expected {E} x {N} contiguous rows")
    if bias.dtype != w.dtype:
        raise UnsupportedValueType(f"bias: operands must share one value type ({bias.dtype}, "
                                   f"{w.dtype})")
    if bias.device != w.device:
        raise _elsewhere(bias, w, "bias")
    return max(N, 1)


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


# ---------------------------------------------------------------- routing

class Routing:
    """The pattern `route` builds: rowptr (E + 1), source (tokens * k: each
    slot's token) and slot (tokens x k: each entry's slot), one index origin."""

    __slots__ = ("rowptr", "source", "slot", "origin")

    def __init__(self, rowptr, source, slot, origin=0):
        self.origin = _origin(origin)
        if slot.dim() != 2:
            raise IncompatibleExtents(f"slot must be tokens x k (got {tuple(slot.shape)})")
        _index(slot, slot.numel(), "slot", slot)
        _index(source, slot.numel(), "source", slot)
        _index(rowptr, rowptr.numel(), "rowptr", slot)
        if rowptr.numel() < 1:
            raise IncompatibleExtents("rowptr must hold experts + 1 positions")
        self.rowptr, self.source, self.slot = rowptr, source, slot

    @property
    def n_experts(self):
        return self.rowptr.numel() - 1

    @property
    def n_slots(self):
        return self.slot.numel()

    def __repr__(self):
        return (f"Routing(tokens={self.slot.shape[0]}, k={self.slot.shape[1]}, "
                f"experts={self.n_experts}, origin={self.origin})")


def route(ids: torch.Tensor, n_experts: int, origin=0) -> Routing:
    """The routing pattern of ids (tokens x k, Int32, origin `origin`): entries
    sorted by expert, in their own order within an expert.  An entry outside
    the experts' range is dropped: it gets no slot (slot = origin - 1)."""
    if ids.dim() != 2:
        raise IncompatibleExtents(f"ids must be tokens x k (got {tuple(ids.shape)})")
    _index(ids, ids.numel(), "ids", ids)
    dev = _on(ids)
    T, k = ids.shape
    E, base = int(n_experts), _base(origin)
    L = _lib.load()
    wsb = L.jlb_route_workspace_size(T, k, E)
    ws = _workspace(wsb, dev)
    slot, source, rowptr = torch.empty_like(ids), ids.new_empty(T * k), ids.new_empty(max(E, 0) + 1)
    st = L.jlb_route(_stream(dev), base, T, k, E, ids.data_ptr(), rowptr.data_ptr(),
                     source.data_ptr(), slot.data_ptr(), _ptr(ws), wsb)
    if st:
        _lib.check(st, "jlb_route")
    r = Routing.__new__(Routing)
    r.rowptr, r.source, r.slot, r.origin = rowptr, source, slot, _origin(origin)
    return r


def _combine_weights(weights, routing, z):
    if weights is None:
        return None
    if weights.dtype != torch.float32:
        raise UnsupportedValueType(f"combine: weights must be Float32 (got {weights.dtype})")
    if weights.shape != routing.slot.shape or not weights.is_contiguous():
        raise IncompatibleExtents(f"combine: weights {tuple(weights.shape)} must be contiguous, "
                                  f"tokens x k = {tuple(routing.slot.shape)}")
    if weights.device != z.device:
        raise _elsewhere(weights, z, "weights")
    return weights


def combine(z: torch.Tensor, routing: Routing, weights=None, out=None) -> torch.Tensor:
    """y[t] = sum_j weights[t, j] * z[slot[t, j]] (weights None: ones), for z
    with a row for every slot; dropped entries add nothing."""
    dt = _type(z, "combine")
    T, k = routing.slot.shape
    S, N = routing.n_slots, z.shape[-1]
    ldz = _rows(z, S, N, "z", z)
    g = _combine_weights(weights, routing, z)
    dev = _on(z)
    if routing.slot.device != dev:
        raise _elsewhere(routing.slot, z, "routing")
    if out is None:
        out = z.new_empty((T, N))
    ldy = _rows(out, T, N, "out", z)
    _lib.call("jlb_combine", _stream(dev), dt, routing.origin.offset, T, k, S, N,
              _ptr(routing.slot), _ptr(g), _ptr(z), ldz, _ptr(out), ldy)
    return out


def combine_backward(dy: torch.Tensor, z: torch.Tensor, routing: Routing, weights=None):
    """Gradients of combine: (dz, dweights), dz[slot[t, j]] = weights[t, j] *
    dy[t] (rows of no slot zero) and dweights[t, j] = <dy[t], z[slot[t, j]]>
    (0 for dropped entries)."""
    dt = _type(z, "combine_backward")
    T, k = routing.slot.shape
    S, N, E = routing.n_slots, z.shape[-1], routing.n_experts
    ldz = _rows(z, S, N, "z", z)
    lddy = _rows(dy, T, N, "dy", z)
    g = _combine_weights(weights, routing, z)
    dev = _on(z)
    if routing.slot.device != dev:
        raise _elsewhere(routing.slot, z, "routing")
    dz = z.new_empty((S, N))
    dg = torch.empty((T, k), dtype=torch.float32, device=dev)
    _lib.call("jlb_combine_backward", _stream(dev), dt, routing.origin.offset, T, k, S, N, E,
              _ptr(routing.rowptr), _ptr(routing.slot), _ptr(g), _ptr(z), ldz, _ptr(dy), lddy,
              _ptr(dz), max(N, 1), _ptr(dg))
    return dz, dg


# ---------------------------------------------------------------- products

def _product(x, w3, rowptr, rows, bias, act, residual, keep_preact, out, base):
    dt = _type(x, "product")
    E, K, N, ldw, sw, order = _weight(w3)
    if w3.dtype != x.dtype:
        raise UnsupportedValueType(f"product: x and w must share one value type ({x.dtype}, "
                                   f"{w3.dtype})")
    dev = _on(x)
    if w3.device != dev:
        raise _elsewhere(w3, x, "w")
    if x.dim() != 2:
        raise IncompatibleExtents(f"x must be a matrix (got {tuple(x.shape)})")
    T = x.shape[0]
    ldx = _rows(x, T, K, "x", x)
    if rowptr is not None:
        _index(rowptr, E + 1, "rowptr", x)
    S = T
    if rows is not None:
        S = rows.numel()
        _index(rows, S, "rows", x)
    ldb = _bias(bias, E, N, x)
    if out is None:
        out = x.new_empty((S, N))
    ldy = _rows(out, S, N, "out", x)
    ldr = _rows(residual, S, N, "residual", x) if residual is not None else 0
    z = x.new_empty((S, N)) if keep_preact else None
    gather = 0 if rows is None else 1
    wsb = _lib.load().jlb_grouped_mm_workspace_size(dt, E, S, T, K, N, _ptr(x), ldx, _ptr(w3), ldw,
                                                    sw, order, gather)
    ws = _workspace(wsb, dev)
    _lib.call("jlb_grouped_mm", _stream(dev), dt, base, E, S, T, K, N, _ptr(rowptr), _ptr(rows),
              _ptr(x), ldx, _ptr(w3), ldw, sw, order, _ptr(bias), ldb, _act(act), _ptr(residual),
              ldr, _ptr(z), max(N, 1), _ptr(out), ldy, _ptr(ws), wsb)
    return (out, z) if keep_preact else out


def grouped_matmul(x, w, rowptr, *, rows=None, bias=None, act=None, keep_preact=False, out=None,
                   origin=0):
    """y[p] = act(x[rows[p]] @ w[e] + bias[e]) for the rows p of group e,
    rowptr[e] .. rowptr[e+1] - 1: x (T x K), w (E x K x N, each matrix row- or
    column-major), rowptr (E + 1, Int32, on the GPU), rows (Int32; None: row p
    of x itself).  Rows past rowptr[E] are zero.  keep_preact returns (y, z)
    with the product before act, which the gradient needs."""
    if rowptr is None:
        raise InvalidArgument("grouped_matmul: rowptr is required")
    return _product(x, _experts(w), rowptr, rows, bias, act, None, keep_preact, out, _base(origin))


def fused_matmul(x, w, *, bias=None, act=None, residual=None, keep_preact=False, out=None):
    """y = act(x @ w + bias) + residual: x (M x K), w (K x N, row- or
    column-major), bias (N), residual (M x N).  keep_preact returns (y, z) with
    the product before act, which the gradient needs.  out may be residual."""
    return _product(x, _dense(w), None, None, bias, act, residual, keep_preact, out, 0)


def _backward(dy, x, w3, rowptr, rows, z, act, need_bias, base):
    dt = _type(x, "product gradient")
    E, K, N, ldw, sw, order = _weight(w3)
    code = _act(act)
    if w3.dtype != x.dtype:
        raise UnsupportedValueType(f"product gradient: x and w must share one value type "
                                   f"({x.dtype}, {w3.dtype})")
    dev = _on(x)
    if w3.device != dev:
        raise _elsewhere(w3, x, "w")
    T = x.shape[0]
    ldx = _rows(x, T, K, "x", x)
    S = T
    if rowptr is not None:
        _index(rowptr, E + 1, "rowptr", x)
    if rows is not None:
        S = rows.numel()
        _index(rows, S, "rows", x)
    lddy = _rows(dy, S, N, "dy", x)
    if code != _lib.ACT_NONE and z is None:
        raise InvalidArgument("product gradient: act needs z, the product before act")
    ldz = _rows(z, S, N, "z", x) if z is not None and code != _lib.ACT_NONE else 0
    L, st = _lib.load(), _stream(dev)
    dz, lddz, db = dy, lddy, None
    if code != _lib.ACT_NONE:
        # dz in the value type: it is an operand of both products, and its
        # rounding enters them like that of any BF16 operand
        lddz = max(8, -(-N // 8) * 8)      # rows that TMA can take as they are
        dz = torch.empty((S, lddz), dtype=x.dtype, device=dev)
    if need_bias:
        db = torch.empty((E, N), dtype=x.dtype, device=dev)
    if need_bias or dz is not dy:
        wsb = L.jlb_act_backward_workspace_size(E, S, N, 1 if need_bias else 0)
        ws = _workspace(wsb, dev)
        _lib.call("jlb_act_backward", st, dt, base, E, S, N, _ptr(rowptr), code, _ptr(dy), lddy,
                  _ptr(z) if ldz else None, ldz, _ptr(dz) if dz is not dy else None, lddz,
                  _ptr(db), max(N, 1), _ptr(ws), wsb)
    # dx = dz W^T: the same product with the weights read in the other order
    dx = torch.empty((S, K), dtype=x.dtype, device=dev)
    wsb = L.jlb_grouped_mm_workspace_size(dt, E, S, S, N, K, _ptr(dz), lddz, _ptr(w3), ldw, sw,
                                          1 - order, 0)
    ws = _workspace(wsb, dev)
    _lib.call("jlb_grouped_mm", st, dt, base, E, S, S, N, K, _ptr(rowptr), None, _ptr(dz), lddz,
              _ptr(w3), ldw, sw, 1 - order, None, 0, 0, None, 0, None, 0, _ptr(dx), max(K, 1),
              _ptr(ws), wsb)
    # dw in w's own order
    if order == _lib.ROW_MAJOR:
        dw, lddw = x.new_empty(w3.shape), max(N, 1)
    else:
        dw = x.new_empty((E, N, K) if w3.dim() == 3 else (N, K)).transpose(-2, -1)
        lddw = max(K, 1)
    gather = 0 if rows is None else 1
    wsb = L.jlb_grouped_mm_wgrad_workspace_size(dt, E, S, T, K, N, _ptr(x), ldx, _ptr(dz), lddz,
                                                order, gather)
    ws = _workspace(wsb, dev)
    _lib.call("jlb_grouped_mm_wgrad", st, dt, base, E, S, T, K, N, _ptr(rowptr), _ptr(rows),
              _ptr(x), ldx, _ptr(dz), lddz, _ptr(dw), lddw, K * N, order, _ptr(ws), wsb)
    return dx, dw, db


def grouped_matmul_backward(dy, x, w, rowptr, *, rows=None, z=None, act=None, bias=False,
                            origin=0):
    """Gradients of grouped_matmul for dy (a row for every output row): (dx,
    dw, db).  With dz = dy * act'(z): dx[p] = dz[p] w[e]^T, one row for every
    output row (with `rows`, a token's gradient is their sum: combine without
    weights); dw[e] = sum of x[rows[p]]^T dz[p], in w's layout; db[e] = sum of
    dz[p] (None unless bias).  With an act, dz is rounded to the value type for
    dx and dw, an operand of two products as dy is (BF16: their relative error
    is 2.3e-3 instead of 1.7e-3); db sums it before that."""
    if rowptr is None:
        raise InvalidArgument("grouped_matmul_backward: rowptr is required")
    return _backward(dy, x, _experts(w), rowptr, rows, z, act, bias, _base(origin))


def fused_matmul_backward(dy, x, w, *, z=None, act=None, bias=False):
    """Gradients of fused_matmul: (dx, dw, db); the residual's is dy itself.  dz =
    dy * act'(z) is rounded to the value type, as in grouped_matmul_backward."""
    dx, dw, db = _backward(dy, x, _dense(w), None, None, z, act, bias, 0)
    return dx, dw, None if db is None else db[0]


# ----------------------------------------------------------------- handles

class B200ProductHandle(AbstractKernelHandle):
    """Prepared product with fixed weights, bias and activation (their buffers
    stay the caller's; values may change): prepare(backend, GroupedMMOp, w,
    bias=, act=, origin=) with w E x K x N, or prepare(backend, FusedMMOp, w,
    bias=, act=) with w K x N."""

    def __init__(self, w, *, grouped, bias=None, act=None, origin=0):
        w3 = _experts(w) if grouped else _dense(w)
        self.dtype = _type(w3, "product")
        self.E, self.K, self.N, ldw, sw, order = _weight(w3)
        self.device = _on(w3)
        self.grouped = grouped
        ldb = _bias(bias, self.E, self.N, w3)
        self.w, self.bias = w3, bias            # keep the buffers alive
        plan = C.c_void_p()
        _lib.call("jlb_mm_plan_create", C.byref(plan), self.dtype, _base(origin), self.E, self.K,
                  self.N, _ptr(w3), ldw, sw, order, _ptr(bias), ldb, _act(act))
        self._plan = plan

    def execute(self, x, rowptr=None, *, rows=None, residual=None, keep_preact=False, out=None):
        """execute(handle, x, rowptr, rows=) of a grouped product, execute(handle,
        x, residual=) of a dense one; as grouped_matmul and fused_matmul."""
        if x.dim() != 2:
            raise IncompatibleExtents(f"x must be a matrix (got {tuple(x.shape)})")
        T, N, w = x.shape[0], self.N, self.w
        ldx = _rows(x, T, self.K, "x", w)
        S = T
        if self.grouped:
            if rowptr is None:
                raise InvalidArgument("grouped product: rowptr is required")
            _index(rowptr, self.E + 1, "rowptr", w)
            if rows is not None:
                S = rows.numel()
                _index(rows, S, "rows", w)
        elif rowptr is not None or rows is not None:
            raise InvalidArgument("a dense product takes no rowptr or rows")
        if out is None:
            out = x.new_empty((S, N))
            ldy = max(N, 1)
        else:
            ldy = _rows(out, S, N, "out", w)
        ldr = _rows(residual, S, N, "residual", w) if residual is not None else 0
        z = x.new_empty((S, N)) if keep_preact else None
        L = _lib.load()
        wsb = L.jlb_mm_plan_workspace_size(self._plan, S, T, _ptr(x), ldx, 0 if rows is None else 1)
        ws = _workspace(wsb, self.device)
        st = L.jlb_mm_plan_execute(self._plan, _stream(self.device), S, T, _ptr(rowptr), _ptr(rows),
                                   _ptr(x), ldx, _ptr(residual), ldr, _ptr(z), max(N, 1), _ptr(out),
                                   ldy, _ptr(ws), wsb)
        if st:
            _lib.check(st, "jlb_mm_plan_execute")
        return (out, z) if keep_preact else out

    def __del__(self):
        try:
            if getattr(self, "_plan", None) and self._plan.value:
                _lib.load().jlb_mm_plan_destroy(self._plan)
                self._plan = C.c_void_p()
        except Exception:
            pass


def execute_product(op_tag, *args, **kw):
    """execute(GroupedMMOp, x, w, rowptr, y, ...) and execute(FusedMMOp, x, w, y, ...):
    in place on y, as the other ops."""
    if op_tag == "GroupedMM":
        x, w, rowptr, y = args
        return grouped_matmul(x, w, rowptr, out=y, **kw)
    x, w, y = args
    return fused_matmul(x, w, out=y, **kw)
