"""Routing, grouped and fused products and their gradients against 64-bit
restatements of their formulas, at the sizes, layouts and values where they
can go wrong."""
import numpy as np
import pytest
import torch

import jlust_b200 as J
import _experts_ref as R
from _helpers import DEV

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
TYPES = [pytest.param(BF, id="bf16"), pytest.param(F32, id="f32")]


def randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def strided(t, extra=0, offset=0):
    """t's values in a buffer with `extra` more elements a row, starting
    `offset` elements in; the rest is NaN."""
    r, c = t.shape
    buf = torch.full((offset + r * (c + extra) + 8,), float("nan"), dtype=t.dtype, device=t.device)
    v = buf[offset:offset + r * (c + extra)].view(r, c + extra)[:, :c]
    v.copy_(t)
    return v


def pointers(sizes, base=0):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64) + base


def dev_i32(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).to(DEV)


def weights(E, K, N, dtype, order, seed):
    w = randn((E, K, N) if order == "row" else (E, N, K), dtype, seed, max(K, 1) ** -0.5)
    return w if order == "row" else w.transpose(1, 2)


# ---------------------------------------------------------------- routing

def random_ids(T, k, E, seed, drop=0.0, base=0):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, E, size=(T, k)) if E else np.zeros((T, k), np.int64)
    if drop:
        ids = np.where(rng.random((T, k)) < drop, rng.choice([-1, E, E + 7, -2 ** 31 + 1]), ids)
    return (ids + base).astype(np.int32)


@pytest.mark.parametrize("T,k,E,drop,base", [
    (0, 4, 8, 0, 0), (1, 1, 1, 0, 0), (1, 8, 8, 0, 1), (5, 3, 2, 0.3, 0), (37, 4, 64, 0, 0),
    (1024, 4, 16, 0, 0), (1023, 4, 300, 0.1, 1), (4097, 1, 7, 0, 0), (2049, 2, 2048, 0, 0),
    (3001, 8, 256, 0.05, 0), (20011, 7, 33, 0.5, 1), (6000, 2, 1500, 0.01, 0), (300, 20, 5, 1.0, 0),
])
def test_route(T, k, E, drop, base):
    ids = random_ids(T, k, E, T + k, drop, base)
    r = J.route(torch.from_numpy(ids).to(DEV), E, origin=base)
    J.device_status()
    rowptr, source, slot = R.route(ids.astype(np.int64), E, base)
    assert np.array_equal(r.rowptr.cpu().numpy(), rowptr)
    assert np.array_equal(r.slot.cpu().numpy(), slot.reshape(T, k))
    assert np.array_equal(r.source.cpu().numpy(), source)


def test_route_of_millions_of_entries():
    """More chunks than a CTA adds up by itself: the counts are scanned."""
    for T, k, E in ((700_001, 2, 19), (400_000, 4, 2048), (40_000, 4, 700)):
        ids = torch.randint(-1, E, (T, k), generator=torch.Generator().manual_seed(E), dtype=torch.int32)
        r = J.route(ids.to(DEV), E, origin=0)
        J.device_status()
        flat = ids.view(-1).long()
        order = torch.sort(torch.where(flat < 0, E, flat), stable=True).indices
        n = int((flat >= 0).sum())
        counts = torch.bincount(flat[flat >= 0], minlength=E)
        assert torch.equal(r.rowptr.cpu().long(), torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]))
        source = torch.full((T * k,), -1, dtype=torch.long)
        source[:n] = order[:n] // k
        slot = torch.full((T * k,), -1, dtype=torch.long)
        slot[order[:n]] = torch.arange(n)
        assert torch.equal(r.source.cpu().long(), source)
        assert torch.equal(r.slot.cpu().long().view(-1), slot)


def test_route_one_expert_takes_all_and_repeats():
    ids = torch.full((9001, 3), 5, dtype=torch.int32, device=DEV)
    a, b = J.route(ids, 9), J.route(ids, 9)
    assert a.rowptr.cpu().tolist() == [0] * 6 + [27003] * 4
    assert torch.equal(a.slot.view(-1), torch.arange(27003, device=DEV, dtype=torch.int32))
    assert torch.equal(a.slot, b.slot) and torch.equal(a.source, b.source)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,N,drop,base,weighted", [
    (1, 1, 1, 0, 0, True), (1, 8, 4096, 0, 0, True), (33, 4, 257, 0.3, 1, True),
    (64, 2, 512, 0, 0, False), (5, 11, 1000, 0.2, 0, True), (700, 3, 96, 1.0, 0, True),
    (0, 2, 8, 0, 0, True), (2000, 8, 40, 0.1, 0, True),
])
def test_combine(dtype, T, k, N, drop, base, weighted):
    E = 13
    r = J.route(torch.from_numpy(random_ids(T, k, E, 3, drop, base)).to(DEV), E, origin=base)
    z = randn((T * k, N), dtype, 1)
    n = int(r.rowptr[-1]) - base
    z[n:] = float("nan")                       # slots of no entry are not read
    g = randn((T, k), F32, 2) if weighted else None
    y = J.combine(z, r, g)
    dy = randn((T, N), dtype, 4)
    dz, dg = J.combine_backward(dy, z, r, g)
    J.device_status()
    slot = r.slot.cpu().numpy().astype(np.int64) - base
    z64, g64, dy64 = R.f64(z), R.f64(g) if weighted else np.ones((T, k)), R.f64(dy)
    ry, by = np.zeros((T, N)), np.zeros((T, N))
    rz, rg, bg = np.zeros((T * k, N)), np.zeros((T, k)), np.zeros((T, k))
    for t in range(T):
        for j in range(k):
            p = slot[t, j]
            if p < 0:
                continue
            ry[t] += g64[t, j] * z64[p]
            by[t] += np.abs(g64[t, j] * z64[p])
            rz[p] = g64[t, j] * dy64[t]
            rg[t, j] = dy64[t] @ z64[p]
            bg[t, j] = np.abs(dy64[t]) @ np.abs(z64[p])
    R.check(y, ry, by * (k + 2) * R.SUM_ULP, dtype, "y")
    R.check(dz, rz, np.abs(rz) * R.SUM_ULP, dtype, "dz")
    R.check(dg, rg, bg * (N + 2) * R.SUM_ULP, F32, "dg")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [1, 40, 129, 1024, 4104])
def test_combine_entries_a_token(dtype, N):
    T, E = 70, 20
    for k in (1, 2, 3, 4, 5, 6, 8, 9):
        ids = random_ids(T, k, E, k, 0.1)
        r = J.route(torch.from_numpy(ids).to(DEV), E)
        z, g, dy = randn((T * k, N), dtype, 1), randn((T, k), F32, 2), randn((T, N), dtype, 4)
        y = J.combine(z, r, g)
        dz, dg = J.combine_backward(dy, z, r, g)
        J.device_status()
        slot = r.slot.cpu().numpy().astype(np.int64)
        live = slot >= 0
        rows = np.where(live[..., None], R.f64(z)[np.maximum(slot, 0)], 0.0)      # T x k x N
        g64, dy64 = R.f64(g), R.f64(dy)
        rz = np.zeros((T * k, N))
        rz[slot[live]] = (g64[..., None] * dy64[:, None])[live]
        R.check(y, np.einsum("tk,tkn->tn", g64, rows),
                np.einsum("tk,tkn->tn", np.abs(g64), np.abs(rows)) * (k + 2) * R.SUM_ULP, dtype, "y")
        R.check(dz, rz, np.abs(rz) * R.SUM_ULP, dtype, "dz")
        R.check(dg, np.einsum("tn,tkn->tk", dy64, rows),
                np.einsum("tn,tkn->tk", np.abs(dy64), np.abs(rows)) * (N + 2) * R.SUM_ULP, F32, "dg")


def test_combine_strided_and_in_place_buffers():
    T, k, N, E = 50, 3, 72, 6
    r = J.route(torch.from_numpy(random_ids(T, k, E, 8)).to(DEV), E)
    z, g = randn((T * k, N), BF, 1), randn((T, k), F32, 2)
    want = J.combine(z, r, g)
    for extra, off in ((8, 0), (3, 0), (8, 1)):
        out = strided(torch.zeros(T, N, dtype=BF, device=DEV), extra, off)
        assert torch.equal(J.combine(strided(z, extra, off), r, g, out=out), want)
        dz, dg = J.combine_backward(strided(want, extra, off), strided(z, extra, off), r, g)
        dz2, dg2 = J.combine_backward(want, z, r, g)
        assert torch.equal(dz, dz2)
        assert (dg - dg2).abs().max() < 1e-4   # another order of the same sums


# ------------------------------------------------------------ the products

GROUPS = {
    "one_row": [1], "decode": [1, 0, 2, 1, 0, 0, 3, 1], "few": [5, 0, 7, 12, 33, 0],
    "mid": [100, 3, 0, 260, 31, 65], "long": [513, 0, 1, 700], "all_empty": [0, 0, 0],
    "many_steps": [1601, 70, 0, 900, 64], "many_experts": [(i * 7) % 5 for i in range(70)],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("groups,K,N,name,base,tail,gather", [
    ("one_row", 256, 512, "gelu", 0, 0, False),
    ("one_row", 1, 1, None, 0, 0, False),
    ("decode", 512, 384, "silu", 0, 2, True),
    ("decode", 1023, 129, "relu", 1, 0, False),
    ("few", 136, 264, "gelu", 0, 5, True),
    ("mid", 320, 640, "silu", 1, 3, True),
    ("mid", 77, 1001, None, 0, 0, False),
    ("long", 192, 256, "gelu", 0, 0, True),
    ("long", 520, 72, "relu", 0, 130, False),
    ("all_empty", 64, 64, None, 0, 9, False),
    ("many_experts", 128, 256, "silu", 0, 0, True),
])
def test_grouped(dtype, order, groups, K, N, name, base, tail, gather):
    sizes = GROUPS[groups]
    E, S = len(sizes), sum(sizes) + tail
    ptr = pointers(sizes)
    T = max(3, S // 2) if gather else S
    rng = np.random.default_rng(K + N)
    rows = rng.integers(0, T, size=S) if gather else None
    x, w = randn((T, K), dtype, 1), weights(E, K, N, dtype, order, 2)
    b = randn((E, N), dtype, 3, 0.5)
    if not gather:
        x[ptr[-1]:] = float("nan")             # rows of no group are not used
    kw = {"rows": None if rows is None else dev_i32(rows + base), "origin": base}
    y, z = J.grouped_matmul(x, w, dev_i32(ptr + base), bias=b, act=name, keep_preact=True, **kw)
    J.device_status()
    x64 = np.nan_to_num(R.f64(x))
    ry, rz, by, bz = R.forward(x64, R.f64(w), ptr, rows, R.f64(b), name)
    ry[ptr[-1]:] = 0
    R.check(z, rz, bz, dtype, "z")
    R.check(y, ry, by, dtype, "y")
    h = J.prepare(J.B200Backend(), J.GroupedMMOp, w, bias=b, act=name, origin=base)
    assert torch.equal(J.execute(h, x, dev_i32(ptr + base), rows=kw["rows"]), y)
    assert torch.equal(J.grouped_matmul(x, w, dev_i32(ptr + base), bias=b, act=name, **kw), y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("groups,K,N,name,base,tail,gather", [
    ("one_row", 64, 128, "silu", 0, 0, False),
    ("decode", 256, 136, "gelu", 1, 2, True),
    ("few", 129, 65, "relu", 0, 0, False),
    ("mid", 320, 256, "silu", 0, 3, True),
    ("mid", 200, 513, None, 1, 70, False),
    ("long", 256, 384, "gelu", 0, 0, False),
    ("all_empty", 32, 48, "relu", 0, 4, False),
    ("many_experts", 64, 72, None, 0, 0, True),
    ("many_steps", 128, 136, None, 0, 0, False),
    ("many_steps", 72, 264, "silu", 0, 5, True),
])
def test_grouped_backward(dtype, order, groups, K, N, name, base, tail, gather):
    sizes = GROUPS[groups]
    E, S = len(sizes), sum(sizes) + tail
    ptr = pointers(sizes)
    T = max(3, S // 2) if gather else S
    rng = np.random.default_rng(K * N)
    rows = rng.integers(0, T, size=S) if gather else None
    x, w = randn((T, K), dtype, 1), weights(E, K, N, dtype, order, 2)
    z, dy = randn((S, N), dtype, 3), randn((S, N), dtype, 4)
    dy[ptr[-1]:] = float("nan")                # rows of no group reach nothing
    z[ptr[-1]:] = float("inf")
    if not gather:
        x[ptr[-1]:] = float("inf")
    dx, dw, db = J.grouped_matmul_backward(dy, x, w, dev_i32(ptr + base), z=z, act=name, bias=True,
                                           rows=None if rows is None else dev_i32(rows + base),
                                           origin=base)
    J.device_status()
    live = ptr[-1]
    dy64, z64, x64 = R.f64(dy), R.f64(z), R.f64(x)
    dy64[live:] = z64[live:] = 0
    if not gather:
        x64[live:] = 0
    ref, bound = R.backward(dy64, x64, R.f64(w), ptr, rows, z64, name, dtype)
    assert dw.stride() == w.contiguous().stride() if order == "row" else dw.stride(1) == 1 or K == 1
    for got, r, b, what in zip((dx, dw, db), ref, bound, ("dx", "dw", "db")):
        R.check(got, r, b, dtype, what)
    again = J.grouped_matmul_backward(dy, x, w, dev_i32(ptr + base), z=z, act=name, bias=True,
                                      rows=None if rows is None else dev_i32(rows + base),
                                      origin=base)
    for a, b in zip(again, (dx, dw, db)):
        assert torch.equal(a, b)               # the same sums in the same order


FUSED = [(1, 256, 512), (1, 4096, 1000), (3, 513, 7), (8, 2048, 640), (16, 1024, 2048),
         (17, 72, 4104), (40, 1000, 384), (128, 64, 128), (130, 640, 257), (257, 96, 520),
         (300, 1536, 264), (2, 1, 3), (5, 8, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("M,K,N", FUSED)
def test_fused(dtype, order, M, K, N):
    name = [None, "relu", "silu", "gelu"][(M + K + N) % 4]
    x, w = randn((M, K), dtype, 1), weights(1, K, N, dtype, order, 2)[0]
    b, r = randn((N,), dtype, 3), randn((M, N), dtype, 4)
    y, z = J.fused_matmul(x, w, bias=b, act=name, residual=r, keep_preact=True)
    J.device_status()
    ry, rz, by, bz = R.forward(R.f64(x), R.f64(w)[None], [0, M], None, R.f64(b)[None], name, R.f64(r))
    R.check(z, rz, bz, dtype, "z")
    R.check(y, ry, by, dtype, "y")
    h = J.prepare(J.B200Backend(), J.FusedMMOp, w, bias=b, act=name)
    assert torch.equal(J.execute(h, x, residual=r), y)
    out = r.clone()
    J.fused_matmul(x, w, bias=b, act=name, residual=out, out=out)      # in place on the residual
    assert torch.equal(out, y)
    # no epilogue at all, through execute
    out = torch.full((M, N), float("nan"), dtype=dtype, device=DEV)
    J.execute(J.FusedMMOp, x, w, out)
    ry, _, by, _ = R.forward(R.f64(x), R.f64(w)[None], [0, M])
    R.check(out, ry, by, dtype, "plain y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("M,K,N,name", [(1, 128, 64, "gelu"), (33, 264, 130, "silu"),
                                        (200, 256, 384, "relu"), (515, 136, 72, None),
                                        (70, 129, 129, "gelu")])
def test_fused_backward(dtype, order, M, K, N, name):
    x, w = randn((M, K), dtype, 1), weights(1, K, N, dtype, order, 2)[0]
    z, dy = randn((M, N), dtype, 3), randn((M, N), dtype, 4)
    dx, dw, db = J.fused_matmul_backward(dy, x, w, z=z, act=name, bias=True)
    J.device_status()
    ref, bound = R.backward(R.f64(dy), R.f64(x), R.f64(w)[None], [0, M], None, R.f64(z), name, dtype)
    R.check(dx, ref[0], bound[0], dtype, "dx")
    R.check(dw, ref[1][0], bound[1][0], dtype, "dw")
    R.check(db, ref[2][0], bound[2][0], dtype, "db")
    dx2, dw2, none = J.fused_matmul_backward(dy, x, w, z=z, act=name)
    assert none is None and torch.equal(dx2, dx) and torch.equal(dw2, dw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [2, 20, 150])
def test_strides_and_misaligned_buffers(dtype, M):
    """Leading dimensions beyond the width and buffers that start between
    16-byte boundaries give the same results; nothing outside is written."""
    K, N = 264, 328
    x, w, r = randn((M, K), dtype, 1), weights(1, K, N, dtype, "row", 2)[0], randn((M, N), dtype, 4)
    b = randn((N,), dtype, 3)
    ry, _, by, _ = R.forward(R.f64(x), R.f64(w)[None], [0, M], None, R.f64(b)[None], "gelu", R.f64(r))
    for extra, off in ((8, 0), (5, 0), (8, 3), (0, 1)):
        out = strided(torch.zeros(M, N, dtype=dtype, device=DEV), extra, off)
        got = J.fused_matmul(strided(x, extra, off), strided(w, extra, off), bias=strided(b[None], 0, off)[0],
                             act="gelu", residual=strided(r, extra, off), out=out)
        J.device_status()
        R.check(got, ry, by, dtype, f"y {extra} {off}")
        if extra:
            pad = torch.as_strided(out, (M - 1, extra), (N + extra, 1), out.storage_offset() + N)
            assert pad.isnan().all()
        wt = strided(w.t().contiguous(), extra, off).t()
        R.check(J.fused_matmul(x, wt, bias=b, act="gelu", residual=r), ry, by, dtype, "col")
        dy = randn((M, N), dtype, 6)
        ref, bound = R.backward(R.f64(dy), R.f64(x), R.f64(w)[None], [0, M], dtype=dtype)
        dx, dw, _ = J.fused_matmul_backward(strided(dy, extra, off), strided(x, extra, off), wt)
        R.check(dx, ref[0], bound[0], dtype, "dx")
        R.check(dw, ref[1][0], bound[1][0], dtype, "dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("K,N", [(96, 136), (97, 133)])
@pytest.mark.parametrize("sizes", [{255: 1}, {0: 1, 256: 2}, {3: 1, 511: 1, 512: 1, 699: 1}, {699: 4},
                                   {0: 9, 300: 18, 640: 1}])
def test_few_rows_among_many_experts(dtype, order, K, N, sizes):
    """The other experts' weights (NaN here) are not used."""
    E = 700
    n = np.zeros(E, np.int64)
    for e, c in sizes.items():
        n[e] = c
    S, ptr = int(n.sum()) + 1, pointers(n)
    x, b = randn((S, K), dtype, 1), randn((E, N), dtype, 3)
    w = torch.full((E, K, N) if order == "row" else (E, N, K), float("nan"), dtype=dtype, device=DEV)
    w = w if order == "row" else w.transpose(1, 2)
    for e in sizes:
        w[e] = randn((K, N), dtype, 10 + e, K ** -0.5)
    y = J.grouped_matmul(x, w, dev_i32(ptr), bias=b, act="silu")
    J.device_status()
    ry, _, by, _ = R.forward(R.f64(x), np.nan_to_num(R.f64(w)), ptr, None, R.f64(b), "silu")
    ry[ptr[-1]:] = 0
    R.check(y, ry, by, dtype, "y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("K,N", [(1024, 264), (1537, 129), (70, 40)])
def test_fused_few_rows(dtype, order, K, N):
    w, b = weights(1, K, N, dtype, order, 2)[0], randn((N,), dtype, 3)
    for M in (1, 2, 3, 4, 5, 8, 9, 16, 17, 24, 25):
        x, res = randn((M, K), dtype, M), randn((M, N), dtype, 5)
        y, z = J.fused_matmul(x, w, bias=b, act="gelu", residual=res, keep_preact=True)
        J.device_status()
        ry, rz, by, bz = R.forward(R.f64(x), R.f64(w)[None], np.array([0, M]), None, R.f64(b)[None],
                                   "gelu", R.f64(res))
        R.check(z, rz, bz, dtype, "z")
        R.check(y, ry, by, dtype, "y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[3, 2], [40, 70, 33], [300, 0, 290]])
def test_bad_values_stay_in_their_rows_and_groups(dtype, sizes):
    """An infinity or NaN in one row reaches that row alone, and a group's dw
    sees only its own rows."""
    E, K, N = len(sizes), 256, 264
    ptr = pointers(sizes)
    S = ptr[-1]
    x, w = randn((S, K), dtype, 1), weights(E, K, N, dtype, "row", 2)
    dy = randn((S, N), dtype, 3)
    clean = J.grouped_matmul(x, w, dev_i32(ptr))
    _, dw_clean, db_clean = J.grouped_matmul_backward(dy, x, w, dev_i32(ptr), bias=True)
    xb, dyb = x.clone(), dy.clone()
    first = ptr[E - 1]                         # the last group's first row
    xb[first, 5], dyb[first, 7] = float("inf"), float("nan")
    got = J.grouped_matmul(xb, w, dev_i32(ptr))
    keep = torch.arange(S, device=DEV) != first
    assert torch.equal(got[keep], clean[keep])
    assert not got[first].isfinite().any()
    _, dw, db = J.grouped_matmul_backward(dyb, xb, w, dev_i32(ptr), bias=True)
    assert torch.equal(dw[:-1], dw_clean[:-1]) and torch.equal(db[:-1], db_clean[:-1])
    assert not dw[-1, 5].isfinite().any() and not dw[-1, :, 7].isfinite().any()
    wb = w.clone()
    wb[0] = float("nan")                       # another expert's weights
    got = J.grouped_matmul(x, wb, dev_i32(ptr))
    assert torch.equal(got[sizes[0]:], clean[sizes[0]:])


def test_relu_keeps_nan_and_lowest_values():
    x = torch.tensor([[float("nan")], [-3.0], [2.0], [torch.finfo(BF).min]], dtype=BF, device=DEV)
    y = J.fused_matmul(x, torch.ones(1, 1, dtype=BF, device=DEV), act="relu").cpu().float().view(-1)
    assert y[0].isnan() and y[1:].tolist() == [0.0, 2.0, 0.0]


def test_row_indices_outside_x_are_reported():
    x, w = randn((4, 64), BF, 1), weights(2, 64, 72, BF, "row", 2)
    rows, ptr = dev_i32([0, 9, 3, -1, 2]), dev_i32([0, 2, 5])
    y = J.grouped_matmul(x, w, ptr, rows=rows)
    with pytest.raises(J.NonCanonicalStorage):
        J.device_status()
    good = J.grouped_matmul(x, w, ptr, rows=dev_i32([0, 0, 3, 0, 2]))
    J.device_status()
    assert torch.equal(y[[0, 2, 4]], good[[0, 2, 4]]) and not y[[1, 3]].any()


def test_row_ranges_outside_the_rows_are_reported():
    x, w = randn((6, 64), BF, 1), weights(3, 64, 72, BF, "row", 2)
    J.grouped_matmul(x, w, dev_i32([0, 4, 2, 9]))
    with pytest.raises(J.NonCanonicalStorage):
        J.device_status()
    J.device_status()


def test_row_ranges_of_late_experts_are_reported():
    x, w = randn((3, 64), F32, 1), weights(400, 64, 72, F32, "row", 2)
    ptr = np.zeros(401, np.int64)
    ptr[350:] = 2
    J.grouped_matmul(x, w, dev_i32(ptr))
    J.device_status()
    ptr[390] = 1                                   # a range that runs backwards
    J.grouped_matmul(x, w, dev_i32(ptr))
    with pytest.raises(J.NonCanonicalStorage):
        J.device_status()
    J.device_status()


def test_offsets_beyond_32_bits():
    """The last expert's weights start past 2^31 elements."""
    E, K, N = 130, 4096, 4104
    w = torch.zeros(E, K, N, dtype=BF, device=DEV)
    assert w.numel() > 2 ** 31
    w[-1] = randn((K, N), BF, 2, K ** -0.5)
    sizes = [0] * (E - 2) + [1, 40]
    ptr = pointers(sizes)
    x = randn((41, K), BF, 1)
    y = J.grouped_matmul(x, w, dev_i32(ptr))
    J.device_status()
    ry, _, by, _ = R.forward(R.f64(x[1:]), R.f64(w[-1:]), [0, 40])
    R.check(y[1:], ry, by, BF, "y")
    assert not y[0].any()
    del y
    dy = randn((41, N), BF, 3)
    dx, dw, _ = J.grouped_matmul_backward(dy, x, w, dev_i32(ptr))
    J.device_status()
    ref, bound = R.backward(R.f64(dy[1:]), R.f64(x[1:]), R.f64(w[-1:]), [0, 40], dtype=BF)
    R.check(dx[1:], ref[0], bound[0], BF, "dx")
    R.check(dw[-1], ref[1][0], bound[1][0], BF, "dw")
    assert not dw[0].any() and not dw[E // 2].any()


def test_another_stream_and_graph_replay():
    E, K, N = 4, 256, 384
    ptr = dev_i32(pointers([9, 0, 30, 5]))
    x, w, b = randn((44, K), BF, 1), weights(E, K, N, BF, "row", 2), randn((E, N), BF, 3)
    want = J.grouped_matmul(x, w, ptr, bias=b, act="silu")
    h = J.prepare(J.B200Backend(), J.GroupedMMOp, w, bias=b, act="silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = J.execute(h, x, ptr)
    s.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        J.execute(h, x, ptr, out=out)
    x.copy_(randn((44, K), BF, 9))
    ptr.copy_(dev_i32(pointers([0, 20, 20, 4])))    # the graph reads the new ranges
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, J.grouped_matmul(x, w, ptr, bias=b, act="silu"))


@pytest.mark.parametrize("name", [None, "relu", "silu", "gelu"])
def test_gradient_against_differences(name):
    """dx, dw, db along random directions against central differences of the
    64-bit forward.  Terms: the differences' own error, h^2 / 6 times a third
    derivative below 2 per unit of |u|^3, and fp32 sums; relu's kinks are kept
    away from the step."""
    sizes, K, N = [7, 0, 12, 1], 24, 18
    E, S, h = len(sizes), sum(sizes), 1e-5
    ptr = pointers(sizes)
    x, w, b = randn((S, K), F32, 1), weights(E, K, N, F32, "row", 2), randn((E, N), F32, 3)
    c = randn((S, N), F32, 4)
    x64, w64, b64, c64 = map(R.f64, (x, w, b, c))
    _, z, _, _ = R.forward(x64, w64, ptr, None, b64, name)
    if name == "relu":
        c64[np.abs(z) < 1e-2] = 0
        c = torch.from_numpy(c64).float().to(DEV)
    y, zk = J.grouped_matmul(x, w, dev_i32(ptr), bias=b, act=name, keep_preact=True)
    grads = J.grouped_matmul_backward(c, x, w, dev_i32(ptr), z=zk, act=name, bias=True)
    rng = np.random.default_rng(5)

    def loss(x_, w_, b_):
        return float((R.forward(x_, w_, ptr, None, b_, name)[0] * c64).sum())

    args = [x64, w64, b64]
    for i, g in enumerate(grads):
        u = rng.standard_normal(args[i].shape)
        plus, minus = list(args), list(args)
        plus[i], minus[i] = args[i] + h * u, args[i] - h * u
        diff = (loss(*plus) - loss(*minus)) / (2 * h)
        g64 = R.f64(g)
        scale = np.abs(g64 * u).sum()
        assert abs((g64 * u).sum() - diff) <= 1e-4 * scale + 1e-6


def test_layer_of_experts_end_to_end():
    """route -> two grouped products -> combine, forward and backward, against
    the layer written per token in 64 bits."""
    T, k, E, D, H = 60, 2, 5, 64, 96
    ids = random_ids(T, k, E, 4)
    ids[:, 1] = (ids[:, 0] + 1) % E
    g = torch.softmax(randn((T, k), F32, 5), 1)
    x, w1, w2 = randn((T, D), F32, 1), weights(E, D, H, F32, "row", 2), weights(E, H, D, F32, "row", 3)
    r = J.route(torch.from_numpy(ids).to(DEV), E)
    h, z = J.grouped_matmul(x, w1, r.rowptr, rows=r.source, act="silu", keep_preact=True)
    o = J.grouped_matmul(h, w2, r.rowptr)
    y = J.combine(o, r, g)
    dy = randn((T, D), F32, 6)
    do, dg = J.combine_backward(dy, o, r, g)
    dh, dw2, _ = J.grouped_matmul_backward(do, h, w2, r.rowptr)
    dxs, dw1, _ = J.grouped_matmul_backward(dh, x, w1, r.rowptr, rows=r.source, z=z, act="silu")
    dx = J.combine(dxs, r)
    J.device_status()
    xt, w1t, w2t, gt = (t.double().cpu().requires_grad_() for t in (x, w1, w2, g))
    out = []
    for t in range(T):
        out.append(sum(gt[t, j] * (torch.nn.functional.silu(xt[t] @ w1t[ids[t, j]]) @ w2t[ids[t, j]])
                       for j in range(k)))
    out = torch.stack(out)
    out.backward(dy.double().cpu())
    # sums of at most a few hundred fp32 terms of order one
    for got, want in ((y, out), (dx, xt.grad), (dw1, w1t.grad), (dw2, w2t.grad), (dg, gt.grad)):
        want = want.detach().numpy()
        assert np.abs(R.f64(got) - want).max() <= 512 * R.SUM_ULP * max(1.0, np.abs(want).max())


@pytest.mark.parametrize("dtype", TYPES)
def test_zero_extents(dtype):
    w, b = weights(3, 8, 16, dtype, "row", 1), randn((3, 16), dtype, 2)
    none = torch.empty(0, 8, dtype=dtype, device=DEV)
    assert J.grouped_matmul(none, w, dev_i32([0, 0, 0, 0]), bias=b).shape == (0, 16)
    dx, dw, db = J.grouped_matmul_backward(torch.empty(0, 16, dtype=dtype, device=DEV), none, w,
                                           dev_i32([0, 0, 0, 0]), bias=True)
    assert dx.shape == (0, 8) and not dw.any() and not db.any()
    # no slots, though x has rows
    x1, no = randn((4, 8), dtype, 3), dev_i32([])
    assert J.grouped_matmul(x1, w, dev_i32([0, 0, 0, 0]), rows=no).shape == (0, 16)
    h = J.prepare(J.B200Backend(), J.GroupedMMOp, w, bias=b)
    assert J.execute(h, x1, dev_i32([0, 0, 0, 0]), rows=no).shape == (0, 16)
    dx, dw, db = J.grouped_matmul_backward(torch.empty(0, 16, dtype=dtype, device=DEV), x1, w,
                                           dev_i32([0, 0, 0, 0]), rows=no, bias=True)
    assert dx.shape == (0, 8) and not dw.any() and not db.any()
    # no inner dimension: the bias alone; no columns: nothing
    x0, w0 = torch.empty(5, 0, dtype=dtype, device=DEV), torch.empty(3, 0, 16, dtype=dtype, device=DEV)
    y = J.grouped_matmul(x0, w0, dev_i32([0, 2, 2, 5]), bias=b, act="relu")
    want = b.clamp_min(0)[[0, 0, 2, 2, 2]]
    assert torch.equal(y, want)
    assert J.fused_matmul(randn((5, 8), dtype, 1), torch.empty(8, 0, dtype=dtype, device=DEV)).shape == (5, 0)
    # every row's index outside x
    y = J.grouped_matmul(none, w, dev_i32([0, 1, 1, 2]), rows=dev_i32([4, -1]))
    with pytest.raises(J.NonCanonicalStorage):
        J.device_status()
    assert not y.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,S,K,N", [(40, 300, 64, 264), (1000, 700, 72, 136), (2, 3000, 512, 64)])
def test_many_groups_and_split_tiles_match_one_group_at_a_time(dtype, E, S, K, N):
    """More groups than a warp looks at together, and tiles split along the
    inner dimension, against the dense product of each group."""
    rng = np.random.default_rng(E)
    cuts = np.sort(rng.integers(0, S + 1, size=E - 1))
    ptr = np.concatenate([[0], cuts, [S]])
    x, w, dy = randn((S, K), dtype, 1), weights(E, K, N, dtype, "row", 2), randn((S, N), dtype, 3)
    y = J.grouped_matmul(x, w, dev_i32(ptr), act="silu")
    dx, dw, db = J.grouped_matmul_backward(dy, x, w, dev_i32(ptr), bias=True)
    J.device_status()
    ry, _, by, _ = R.forward(R.f64(x), R.f64(w), ptr, name="silu")
    ref, bound = R.backward(R.f64(dy), R.f64(x), R.f64(w), ptr, dtype=dtype)
    R.check(y, ry, by, dtype, "y")
    for got, r, b, what in zip((dx, dw, db), ref, bound, ("dx", "dw", "db")):
        R.check(got, r, b, dtype, what)


@pytest.mark.parametrize("dtype", TYPES)
def test_graph_of_a_training_step(dtype):
    """route, the products (few tiles, so split ones too), combine and every
    gradient captured once and replayed on new values."""
    T, k, E, D, H = 333, 2, 4, 512, 264
    ids = dev_i32(random_ids(T, k, E, 4))
    x, w = randn((T, D), dtype, 1), weights(E, D, H, dtype, "row", 2)
    g, dy = torch.softmax(randn((T, k), F32, 5), 1), randn((T, H), dtype, 6)

    def step():
        r = J.route(ids, E)
        y, z = J.grouped_matmul(x, w, r.rowptr, rows=r.source, act="gelu", keep_preact=True)
        out = J.combine(y, r, g)
        do, dg = J.combine_backward(dy, y, r, g)
        dxs, dw, db = J.grouped_matmul_backward(do, x, w, r.rowptr, rows=r.source, z=z, act="gelu",
                                                bias=True)
        return out, dg, J.combine(dxs, r), dw, db

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    ids.copy_(dev_i32(random_ids(T, k, E, 9, 0.2)))
    x.copy_(randn((T, D), dtype, 11))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(kept, step()):
        assert torch.equal(a, b)
    J.device_status()


@pytest.mark.parametrize("M,K,N", [(20, 256, 64), (200, 512, 264), (4, 128, 96)])
def test_f32_infinities_and_large_values_keep_their_places(M, K, N):
    """F32 runs as planes of bf16: an infinity, a NaN or a value near the
    type's largest gives what the products and sums of fp32 give."""
    x, w = randn((M, K), F32, 1), randn((K, N), F32, 2, K ** -0.5)
    inf = float("inf")
    x[0, 3], x[1, 4], x[1, 5], x[2, 6] = inf, inf, -inf, float("nan")
    w[3, 1], w[3, 2], w[7, 3], w[8, 4] = 0.0, -inf, inf, float("nan")
    x[3, 9], w[9, :] = 3.4028e38, 1e-3
    y, want = J.fused_matmul(x, w).cpu(), (x.cpu().double() @ w.cpu().double())
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y.isinf(), want.isinf()) and torch.equal(y[y.isinf()].sign(), want[want.isinf()].sign())
    ok = want.isfinite()
    scale = (x.cpu().double().abs().nan_to_num(0, 0, 0) @ w.cpu().double().abs().nan_to_num(0, 0, 0))
    assert ((y - want).abs()[ok] <= (K + 8) * R.SUM_ULP * scale[ok] + 1e-37).all()
