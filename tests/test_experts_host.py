"""The expert-layer operators refuse what they cannot run, with the
framework's own errors, before any device work."""
import ctypes as C

import pytest
import torch

import jlust_b200 as J
from jlust_b200 import _lib

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def t(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,error", [
    (lambda: J.route(t(4, dtype=I32), 4), J.IncompatibleExtents),
    (lambda: J.route(t(4, 2, dtype=torch.int64), 4), J.UnsupportedIndexType),
    (lambda: J.route(t(4, 2, dtype=I32), 4), J.DeviceMismatch),
    (lambda: J.route(t(4, 4, dtype=I32)[:, :2], 4), J.IncompatibleExtents),
    (lambda: J.grouped_matmul(t(4, 8), t(2, 8, 6), t(3, dtype=I32)), J.DeviceMismatch),
    (lambda: J.grouped_matmul(t(4, 8), t(2, 8, 6), None), J.errors.InvalidArgument),
    (lambda: J.grouped_matmul(t(4, 8, dtype=torch.float64), t(2, 8, 6, dtype=torch.float64),
                              t(3, dtype=I32)), J.UnsupportedValueType),
    (lambda: J.grouped_matmul(t(4, 8), t(2, 8, 6, dtype=F32), t(3, dtype=I32)),
     J.UnsupportedValueType),
    (lambda: J.fused_matmul(t(4, 8), t(2, 8, 6)), J.IncompatibleExtents),
    (lambda: J.fused_matmul(t(4, 8), t(16, 12)[::2, ::2]), J.IncompatibleExtents),
    (lambda: J.fused_matmul_backward(t(4, 6), t(4, 8), t(8, 6), act="tanh"),
     J.errors.InvalidArgument),
    (lambda: J.fused_matmul_backward(t(4, 6), t(4, 8), t(1, 8, 6)), J.IncompatibleExtents),
    (lambda: J.grouped_matmul_backward(t(4, 6), t(4, 8), t(2, 8, 6), None),
     J.errors.InvalidArgument),
    (lambda: J.prepare(J.B200Backend(), J.FusedMMOp, t(8, 6)), J.DeviceMismatch),
    (lambda: J.prepare(J.B200Backend(), J.FusedMMOp, t(2, 8, 6)), J.IncompatibleExtents),
    (lambda: J.Routing(t(3, dtype=I32), t(5, dtype=I32), t(3, 2, dtype=I32)),
     J.IncompatibleExtents),
    (lambda: J.combine(t(6, 4), J.Routing(t(3, dtype=I32), t(6, dtype=I32), t(3, 2, dtype=I32))),
     J.DeviceMismatch),
    (lambda: J.combine(t(5, 4), J.Routing(t(3, dtype=I32), t(6, dtype=I32), t(3, 2, dtype=I32))),
     J.IncompatibleExtents),
    (lambda: J.combine(t(6, 4), J.Routing(t(3, dtype=I32), t(6, dtype=I32), t(3, 2, dtype=I32)),
                       t(3, 2)), J.UnsupportedValueType),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def test_supports_backend():
    be, D = J.B200Backend(), J.Formats.DensedRight
    assert J.supports_backend(be, J.GroupedMMOp(D(2), D(3), D(1), D(2)))
    assert J.supports_backend(be, J.FusedMMOp(D(2), D(2), D(2)))
    assert not J.supports_backend(be, J.GroupedMMOp(D(2), D(2), D(1), D(2)))
    assert not J.supports_backend(be, J.FusedMMOp(J.Formats.CSR, D(2), D(2)))


P = C.c_void_p(4096)     # never dereferenced: every call below is refused first


def _mm(**kw):
    a = dict(stream=None, dtype=2, base=0, E=2, S=4, T=4, K=8, N=16, rowptr=P, rows=None, x=P, ldx=8,
             w=P, ldw=16, sw=128, order=0, bias=None, ldb=0, act=0, res=None, ldr=0, z=None, ldz=0,
             y=P, ldy=16, ws=None, wsb=0)
    a.update(kw)
    return _lib.load().jlb_grouped_mm(*a.values())


@pytest.mark.parametrize("kw,status", [
    ({"dtype": 1}, 3), ({"dtype": 9}, 3), ({"base": 2}, 8), ({"E": -1}, 6), ({"S": -4}, 6),
    ({"K": -1}, 6), ({"act": 4}, 8), ({"act": -1}, 8), ({"order": 2}, 8), ({"ldw": 15}, 6),
    ({"ldx": 7}, 6), ({"ldy": 15}, 6), ({"sw": 100}, 6), ({"rowptr": None}, 8), ({"T": 5}, 6),
    ({"x": None}, 8), ({"w": None}, 8), ({"y": None}, 8), ({"S": 2 ** 31, "T": 2 ** 31}, 2),
    ({"E": 0}, 6), ({"res": P, "ldr": 3}, 6), ({"z": P, "ldz": 3}, 6), ({"bias": P, "ldb": 3}, 6),
])
def test_product_statuses(kw, status):
    assert _mm(**kw) == status
    assert len(_lib.last_error()) > 0


def test_size_queries_take_any_extents():
    L = _lib.load()
    for bad in (-1, -40, -2 ** 40):
        for i in range(5):                      # E, S, T, K, N
            a = [2, 64, 64, 64, 64]
            a[i] = bad
            assert L.jlb_grouped_mm_workspace_size(2, *a, P, 64, P, 64, 4096, 0, 0) == 0
            assert L.jlb_grouped_mm_wgrad_workspace_size(2, *a, P, 64, P, 64, 0, 0) == 0
    for a in ((0, 5, 5, 8, 8), (3, 0, 0, 8, 8), (3, 5, 5, 0, 8), (3, 5, 5, 8, 0), (3, 5, 0, 8, 8)):
        for dtype in (0, 2):
            L.jlb_grouped_mm_workspace_size(dtype, *a, P, 8, P, 8, 64, 0, 0)
            L.jlb_grouped_mm_wgrad_workspace_size(dtype, *a, P, 8, P, 8, 0, 0)
    assert L.jlb_act_backward_workspace_size(-1, 5, 8, 1) == 0
    assert L.jlb_route_workspace_size(-1, 5, 8) == 0


def test_other_statuses():
    L = _lib.load()
    assert L.jlb_route(None, 0, 4, 2, 4096, P, P, P, P, None, 0) == 1          # too many experts
    assert L.jlb_route(None, 0, 2 ** 30, 4, 8, P, P, P, P, None, 0) == 2
    assert L.jlb_route(None, 0, 10000, 4, 8, P, P, P, P, None, 0) == 11        # workspace
    assert L.jlb_route(None, 3, 4, 2, 8, P, P, P, P, None, 0) == 8
    assert L.jlb_route(None, 0, 4, 2, 8, None, P, P, P, None, 0) == 8
    assert L.jlb_route_workspace_size(10000, 4, 8) > 0 == L.jlb_route_workspace_size(4, 2, 8)
    assert L.jlb_combine(None, 1, 0, 4, 2, 8, 16, P, P, P, 16, P, 16) == 3
    assert L.jlb_combine(None, 2, 0, 4, 2, 8, 16, P, P, P, 15, P, 16) == 6
    assert L.jlb_combine(None, 2, 0, 4, 2, 8, 16, None, P, P, 16, P, 16) == 8
    assert L.jlb_combine_backward(None, 2, 0, 4, 2, 8, 16, 3, None, P, P, P, 16, P, 16, P, 16, P) == 8
    assert L.jlb_grouped_mm_wgrad(None, 2, 0, 2, 4, 4, 8, 16, P, None, P, 8, P, 15, P, 16, 128, 0,
                                  None, 0) == 6
    assert L.jlb_grouped_mm_wgrad(None, 2, 0, 2, 4, 4, 8, 16, P, None, P, 8, P, 16, None, 16, 128, 0,
                                  None, 0) == 8
    assert L.jlb_act_backward(None, 2, 0, 2, 4, 16, P, 1, P, 16, None, 0, P, 16, P, 16, None, 0) == 8
    assert L.jlb_act_backward(None, 2, 0, 2, 4, 16, P, 0, P, 16, None, 0, None, 0, P, 16, None, 0) == 11
    h = C.c_void_p()
    assert L.jlb_mm_plan_create(C.byref(h), 1, 0, 2, 8, 16, P, 16, 128, 0, None, 0, 0) == 3
    assert not h.value
    assert L.jlb_mm_plan_execute(None, None, 4, 4, P, None, P, 8, None, 0, None, 0, P, 16, None, 0) == 8
    assert L.jlb_mm_plan_destroy(None) == 0
