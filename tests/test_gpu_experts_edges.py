"""Expert-layer operators at the edges of their contracts: row ranges that
overlap, tails of the activations, extents past a launch's limits, and what
has to be waited for before a kernel ends."""
import math

import numpy as np
import pytest
import torch

import jlust_b200 as J
import _experts_ref as R
from _planes import F32_NORM
from _helpers import DEV
from jlust_b200 import _lib

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
TYPES = [pytest.param(BF, id="bf16"), pytest.param(F32, id="f32")]


def randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def dev_i32(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).to(DEV)


# ------------------------------------------------- row ranges that overlap

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [40, 41])
def test_bias_sums_of_overlapping_ranges_stay_in_their_workspace(dtype, N):
    """rowptr [0, S, 0, S, ...] gives every second group all rows: more row
    tiles than the workspace has parts.  Past its bytes lies NaN, which no sum
    may read; the first group's sums are those of its rows."""
    L, S, E = _lib.load(), 1000, 9
    dy, ptr = randn((S, N), dtype, 1), dev_i32([0, S] * 5)
    wsb = L.jlb_act_backward_workspace_size(E, S, N, 1)
    ws = torch.full((wsb // 4 + 64 * N,), float("nan"), device=DEV)
    db = torch.full((E, N), float("nan"), dtype=dtype, device=DEV)
    st = L.jlb_act_backward(torch.cuda.current_stream().cuda_stream, 0 if dtype == F32 else 2, 0, E, S, N,
                            ptr.data_ptr(), 0, dy.data_ptr(), N, None, 0, None, 0, db.data_ptr(), N,
                            ws.data_ptr(), wsb)
    assert st == 0
    with pytest.raises(J.NonCanonicalStorage):
        J.device_status()
    J.device_status()
    assert db.isfinite().all() and not db[1].any()
    dy64 = R.f64(dy)
    R.check(db[0], dy64.sum(0), (S + 8) * R.SUM_ULP * np.abs(dy64).sum(0), dtype, "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ptr", [[0, 300, 0, 300], [0, 40, 20, 300], [5, 60, 400, 200], [0, 100, 200, -7]])
def test_gradients_report_bad_ranges(dtype, ptr):
    E, S, K, N = len(ptr) - 1, 300, 72, 136
    x, w, z, dy = randn((S, K), dtype, 1), randn((E, K, N), dtype, 2), randn((S, N), dtype, 3), randn((S, N), dtype, 4)
    for act in (None, "silu"):
        J.grouped_matmul_backward(dy, x, w, dev_i32(ptr), z=z, act=act, bias=True)
        with pytest.raises(J.NonCanonicalStorage):
            J.device_status()
        J.device_status()


# --------------------------------------- what a launch waits for at its end

@pytest.mark.parametrize("dtype", TYPES)
def test_products_back_to_back_with_few_and_many_tiles_a_pair(dtype):
    """One, two, three and more tiles a CTA pair (each accumulator's last use
    odd or even), empty groups, and tiles drawn from the counter with fewer and
    more tickets than places: a launch that waited for an arrival that does not
    come would report a timeout, and the next ones repeat its results."""
    K, N = 128, 512
    for sizes in ([300], [0, 40], [300] * 40, [0, 900, 33] * 50, [1] * 80, [256] * 300):
        ptr, E, S = dev_i32(np.concatenate([[0], np.cumsum(sizes)])), len(sizes), sum(sizes)
        x, w, dy = randn((S, K), dtype, 1), randn((E, K, N), dtype, 2), randn((S, N), dtype, 3)
        first = None
        for _ in range(20):
            got = (J.grouped_matmul(x, w, ptr), *J.grouped_matmul_backward(dy, x, w, ptr)[:2])
            first = first or got
        J.device_status()
        assert all(torch.equal(a, b) for a, b in zip(got, first))


# -------------------------------------------------- tails of the activations

def tail(dtype, M):
    z = torch.linspace(-10, -3, M, dtype=torch.float64).to(dtype)
    return z.view(M, 1).to(DEV), z.double().numpy()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [8, 40, 700])
def test_gelu_keeps_its_negative_tail(dtype, M):
    """Relative to the result, value and slope, against erfc in 64 bits.  F32:
    the argument z / sqrt 2 is rounded twice (a unit and a half of 2^-24), which
    erfc multiplies by z^2 + 1; erfcf's 4 units and the products' roundings are
    a dozen more.  In the slope expf(-z^2 / 2) does the same and the difference
    of the two terms is 0.8 of the larger at least.  BF16: 5e-6 of the fit, and
    the same with the cheaper exponential's 60 units of 2^-23, below 1e-4 in
    all, then the rounding."""
    z, z64 = tail(dtype, M)
    phi = np.array([0.5 * math.erfc(-v / math.sqrt(2)) for v in z64])
    slope = phi + z64 * np.exp(-0.5 * z64 * z64) / math.sqrt(2 * math.pi)
    one = torch.ones(1, 1, dtype=dtype, device=DEV)
    y = J.fused_matmul(z, one, act="gelu")
    dz, _, _ = J.fused_matmul_backward(torch.ones_like(z), z, one, z=z, act="gelu")
    J.device_status()
    rel = (3 * z64 * z64 + 32) * 2.0 ** -24 if dtype == F32 else 1e-4
    for got, want in ((y, z64 * phi), (dz, slope)):
        err = np.abs(R.f64(got)[:, 0] / want - 1)
        lim = rel + R.HALF_ULP[dtype] * (1 + rel)
        assert (err <= lim).all(), (z64[err > lim][0], err.max())


# ------------------------------------------------ how exact F32 products are

@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("K,N", [(320, 640), (520, 257), (1536, 264), (641, 72)])
@pytest.mark.parametrize("sizes", [[130], [459], [260, 31, 0, 168], [1601, 70]])
def test_f32_products_keep_three_planes(order, K, N, sizes):
    """The forward product, dx and dw of shapes that run as planes of bf16, in
    the norm: element by element, a bound for any values lets a lost third
    plane through."""
    ptr, E, S = np.concatenate([[0], np.cumsum(sizes)]), len(sizes), sum(sizes)
    x, dy = randn((S, K), F32, 1), randn((S, N), F32, 3)
    w = randn((E, K, N), F32, 2) if order == "row" else randn((E, N, K), F32, 2).transpose(1, 2)
    y = J.grouped_matmul(x, w, dev_i32(ptr))
    dx, dw, _ = J.grouped_matmul_backward(dy, x, w, dev_i32(ptr))
    J.device_status()
    ry, _, _, _ = R.forward(R.f64(x), R.f64(w), ptr)
    (rdx, rdw, _), _ = R.backward(R.f64(dy), R.f64(x), R.f64(w), ptr)
    for got, want, what in ((y, ry, "y"), (dx, rdx, "dx"), (dw, rdw, "dw")):
        assert np.linalg.norm(R.f64(got) - want) <= F32_NORM * np.linalg.norm(want), what
    if E == 1:
        y = J.fused_matmul(x, w[0])
        assert np.linalg.norm(R.f64(y) - ry) <= F32_NORM * np.linalg.norm(ry)


# ------------------------------------------ extents past a launch's y and z

def test_bias_sums_of_overlapping_ranges_past_the_grid():
    """More tiles than grid y holds and ranges that overlap: the grid's last
    layer has no part to write."""
    L, S, E, N = _lib.load(), 65535 * 128 + 300, 3, 8
    dy, ptr = torch.ones(S, N, dtype=BF, device=DEV), dev_i32([0, S, 0, S])
    wsb = L.jlb_act_backward_workspace_size(E, S, N, 1)
    ws = torch.full((wsb // 4 + (1 << 22),), float("nan"), device=DEV)
    db = torch.empty(E, N, dtype=BF, device=DEV)
    assert L.jlb_act_backward(torch.cuda.current_stream().cuda_stream, 2, 0, E, S, N, ptr.data_ptr(), 0,
                              dy.data_ptr(), N, None, 0, None, 0, db.data_ptr(), N, ws.data_ptr(), wsb) == 0
    with pytest.raises(J.NonCanonicalStorage):
        J.device_status()
    J.device_status()
    assert ws[wsb // 4:].isnan().all() and db.isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_more_rows_than_a_grid_has_tiles(dtype):
    """65,535 tiles of 128 rows and more.  Ones in the last rows: their sums
    are whole numbers, exact in either type."""
    S, N, tail = 65535 * 128 + 300, 8, 200
    dy, x = torch.zeros(S, N, dtype=dtype, device=DEV), torch.ones(S, N, dtype=dtype, device=DEV)
    dy[-tail:] = 1
    w = torch.eye(N, dtype=dtype, device=DEV)
    for act in (None, "relu"):
        assert J.fused_matmul(x, w, act=act).shape == (S, N)
        dx, dw, db = J.fused_matmul_backward(dy, x, w, z=x, act=act, bias=True)
        J.device_status()
        assert torch.equal(dx, dy)
        assert torch.equal(db, torch.full_like(db, tail)) and torch.equal(dw, torch.full_like(dw, tail))


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_more_experts_than_a_grid_has_rows(dtype):
    E, N = 70_000, 8
    n = np.zeros(E, np.int64)
    n[[3, 65_534, 65_535, 65_536, E - 1]] = [5, 2, 7, 1, 4]
    ptr, S = dev_i32(np.concatenate([[0], np.cumsum(n)])), int(n.sum())
    x, w = torch.ones(S, N, dtype=dtype, device=DEV), torch.ones(E, N, N, dtype=dtype, device=DEV)
    z, dy = torch.ones_like(x), torch.ones_like(x)
    y = J.grouped_matmul(x, w, ptr)
    dx, dw, db = J.grouped_matmul_backward(dy, x, w, ptr, z=z, act="relu", bias=True)
    J.device_status()
    assert torch.equal(y, torch.full_like(y, N)) and torch.equal(dx, torch.full_like(dx, N))
    want = torch.from_numpy(n).to(DEV).to(dtype)
    assert torch.equal(db, want[:, None].expand(E, N)) and torch.equal(dw, want[:, None, None].expand(E, N, N))
    # no rows at all: zeros
    none = torch.empty(0, N, dtype=dtype, device=DEV)
    dx, dw, db = J.grouped_matmul_backward(none, none, w, torch.zeros_like(ptr), bias=True)
    J.device_status()
    assert dx.shape == (0, N) and not dw.any() and not db.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_products_without_an_inner_dimension_of_many_rows(dtype):
    S, N = 65535 * 128 + 300, 8
    b = randn((N,), dtype, 1)
    y = J.fused_matmul(torch.empty(S, 0, dtype=dtype, device=DEV), torch.empty(0, N, dtype=dtype, device=DEV), bias=b)
    J.device_status()
    assert torch.equal(y, b.expand(S, N))


# ------------------------------------------- routing around its two ways

@pytest.mark.parametrize("E,chunks", [(512, 127), (512, 128), (16, 512), (64, 341), (64, 342), (128, 255), (128, 256),
                                      (2048, 31), (2048, 32), (1, 600)])
def test_route_on_both_sides_of_scanning_its_counts(E, chunks):
    """4096 entries a chunk, the last one short."""
    n = chunks * 4096 - 1000
    ids = torch.randint(-1, E + 1, (n, 1), generator=torch.Generator().manual_seed(E + chunks), dtype=torch.int32)
    r = J.route(ids.to(DEV), E)
    J.device_status()
    flat = ids.view(-1).long()
    key = torch.where((flat < 0) | (flat >= E), E, flat)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=E + 1)[:E]
    live = int(counts.sum())
    assert torch.equal(r.rowptr.cpu().long(), torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]))
    slot = torch.full((n,), -1, dtype=torch.long)
    slot[order[:live]] = torch.arange(live)
    source = torch.full((n,), -1, dtype=torch.long)
    source[:live] = order[:live]
    assert torch.equal(r.slot.cpu().long().view(-1), slot) and torch.equal(r.source.cpu().long(), source)


# ------------------------------------------------------------ entry points

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["row", "col"])
def test_execute_grouped_in_place(dtype, order):
    """execute(GroupedMMOp, x, w, rowptr, y, ...) writes y as grouped_matmul
    returns it."""
    E, K, N, sizes, base = 3, 72, 136, [40, 0, 25], 1
    ptr, S = dev_i32(np.concatenate([[0], np.cumsum(sizes)]) + base), sum(sizes)
    w = randn((E, K, N), dtype, 2) if order == "row" else randn((E, N, K), dtype, 2).transpose(1, 2)
    x, b = randn((S, K), dtype, 1), randn((E, N), dtype, 3)
    rows = dev_i32(np.random.default_rng(4).integers(0, S, S) + base)
    y = torch.full((S, N), float("nan"), dtype=dtype, device=DEV)
    J.execute(J.GroupedMMOp, x, w, ptr, y, bias=b, act="silu", rows=rows, origin=base)
    J.device_status()
    assert torch.equal(y, J.grouped_matmul(x, w, ptr, bias=b, act="silu", rows=rows, origin=base))
    with pytest.raises(J.IncompatibleExtents):
        J.execute(J.GroupedMMOp, x, w, ptr, y[:-1], origin=base)
    with pytest.raises(J.UnsupportedIndexType):
        J.execute(J.GroupedMMOp, x, w, ptr.long(), y, origin=base)
