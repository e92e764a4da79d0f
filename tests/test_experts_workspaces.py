"""The expert-layer entry points refuse a workspace that is missing, short or not
16-byte aligned before any device work."""
import ctypes as C

import pytest

from jlust_b200 import _lib

P = 4096                                # never dereferenced
NEED = {
    "route": lambda L: L.jlb_route_workspace_size(10000, 4, 8),
    "product": lambda L: L.jlb_grouped_mm_workspace_size(2, 2, 100, 100, 9, 16, P, 9, P, 16, 144, 0, 0),
    "gradient": lambda L: L.jlb_grouped_mm_wgrad_workspace_size(2, 2, 100, 100, 9, 16, P, 9, P, 16, 0, 0),
    "act": lambda L: L.jlb_act_backward_workspace_size(2, 100, 16, 1),
}
CALL = {
    "route": lambda L, ws, n: L.jlb_route(None, 0, 10000, 4, 8, P, P, P, P, ws, n),
    "product": lambda L, ws, n: L.jlb_grouped_mm(None, 2, 0, 2, 100, 100, 9, 16, P, None, P, 9, P, 16, 144, 0, None,
                                                 0, 0, None, 0, None, 0, P, 16, ws, n),
    "gradient": lambda L, ws, n: L.jlb_grouped_mm_wgrad(None, 2, 0, 2, 100, 100, 9, 16, P, None, P, 9, P, 16, P, 16,
                                                        144, 0, ws, n),
    "act": lambda L, ws, n: L.jlb_act_backward(None, 2, 0, 2, 100, 16, P, 0, P, 16, None, 0, None, 0, P, 16, ws, n),
}


@pytest.mark.parametrize("name", sorted(CALL))
def test_workspaces(name):
    L = _lib.load()
    need = NEED[name](L)
    assert need > 0
    for ws, n in ((None, need), (P, need - 1), (P + 4, need), (P + 8, need), (P + 1, need)):
        assert CALL[name](L, C.c_void_p(ws), C.c_size_t(n)) == 11, (ws, n)
        assert "16-byte aligned" in _lib.last_error()
