"""Graph captures are not disturbed by Python's garbage."""
import gc

import pytest
import torch

import jlust_b200 as J

pytestmark = pytest.mark.gpu


def test_no_cyclic_collection_during_a_block_product_capture():
    n, dev = 8, "cuda"
    ptr = torch.arange(n + 1, dtype=torch.int32, device=dev)
    block = J.csr_tensor(ptr, ptr[:n].clone(), torch.arange(1.0, n + 1, dtype=torch.float64, device=dev), (n, n),
                         origin=0)
    A = J.BlockSparseMatrix([[block]])
    x = torch.rand(n, dtype=torch.float64, device=dev)
    y = torch.zeros(n, dtype=torch.float64, device=dev)
    J.mul(y, A, x)
    run, seen = A._compiled.spmv, []

    def spmv(x, y):
        seen.append((torch.cuda.is_current_stream_capturing(), gc.isenabled()))
        run(x, y)

    A._compiled.spmv = spmv
    y2 = torch.zeros_like(y)
    for enabled in (True, False):
        A._compiled.graphs.clear()
        (gc.enable if enabled else gc.disable)()
        try:
            J.mul(y2, A, x)
            assert gc.isenabled() == enabled
        finally:
            gc.enable()
    assert (True, False) in seen and (True, True) not in seen
    J.device_status()
    assert torch.equal(y, y2) and torch.equal(y, x * torch.arange(1.0, n + 1, dtype=torch.float64, device=dev))
