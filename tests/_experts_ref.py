"""The expert-layer operators in 64 bits on the host, straight from their
formulas, and the error bounds the tests hold the kernels to."""
import math

import numpy as np
import torch

# unit roundoff of a value type (round to nearest: 2^-p for p significant bits, 8
# and 24), and of the fp32 sums: a tensor-core sum may truncate, so a whole
# unit of 2^-23 a term
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SUM_ULP = 2.0 ** -23


def act(z, name):
    if name == "relu":
        return np.where(z < 0, 0.0, z)
    if name == "silu":
        return z / (1 + np.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + np.vectorize(math.erf, otypes=[float])(z / math.sqrt(2)))
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).astype(np.float64)
    if name == "silu":
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return (0.5 * (1 + np.vectorize(math.erf, otypes=[float])(z / math.sqrt(2)))
                + z * np.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    return np.ones_like(z)


def f64(t):
    return None if t is None else t.detach().cpu().double().numpy()


def route(ids, E, base=0):
    """rowptr, source, slot by a plain loop over the entries."""
    T, k = ids.shape
    rowptr = np.zeros(E + 1, np.int64)
    slot = np.full((T, k), -1, np.int64)
    source = np.full(T * k, -1, np.int64)
    for e in range(E):
        p = rowptr[e]
        for t, j in np.argwhere(ids - base == e):
            slot[t, j], source[p] = p, t
            p += 1
        rowptr[e + 1] = p
    return rowptr + base, source + base, slot + base


def forward(x, w, rowptr, rows=None, bias=None, name=None, res=None):
    """(y, z, bound of y, bound of z): the bounds hold everything but the last
    rounding -- one unit of 2^-23 of sum |x||w| a term, passed through act,
    whose slope stays within 1.13, and a few units for act itself."""
    S = rows.shape[0] if rows is not None else x.shape[0]
    E, K, N = w.shape
    y, z = np.zeros((S, N)), np.zeros((S, N))
    by, bz = np.zeros((S, N)), np.zeros((S, N))
    for e in range(E):
        a, b = rowptr[e], rowptr[e + 1]
        xe = x[rows[a:b]] if rows is not None else x[a:b]
        z[a:b] = xe @ w[e]
        bz[a:b] = np.abs(xe) @ np.abs(w[e])
        if bias is not None:
            z[a:b] += bias[e]
            bz[a:b] += np.abs(bias[e])
        y[a:b] = act(z[a:b], name)
    bz *= (K + 8) * SUM_ULP
    by = 1.13 * bz + 64 * SUM_ULP * np.abs(z)
    if res is not None:
        y += res
        by += SUM_ULP * np.abs(y)
    return y, z, by, bz


def backward(dy, x, w, rowptr, rows=None, z=None, name=None, dtype=torch.float32):
    """(dx, dw, db) and their bounds; dz is an operand in the value type, so
    its rounding enters dx and dw."""
    S, (E, K, N) = dy.shape[0], w.shape
    dz = dy * slope(z, name) if name not in (None, "none") else dy
    # rounding of dz, and act' itself: a few fp32 units of values around one
    rz = (HALF_ULP[dtype] * np.abs(dz) + 64 * SUM_ULP * np.abs(dy)) if dz is not dy else 0 * dy
    dx, bx = np.zeros((S, K)), np.zeros((S, K))
    dw, bw = np.zeros((E, K, N)), np.zeros((E, K, N))
    db, bb = np.zeros((E, N)), np.zeros((E, N))
    for e in range(E):
        a, b = rowptr[e], rowptr[e + 1]
        xe = x[rows[a:b]] if rows is not None else x[a:b]
        d, r = dz[a:b], rz[a:b]
        dx[a:b] = d @ w[e].T
        bx[a:b] = (r + (N + 8) * SUM_ULP * np.abs(d)) @ np.abs(w[e]).T
        dw[e] = xe.T @ d
        bw[e] = np.abs(xe).T @ (r + (b - a + 8) * SUM_ULP * np.abs(d))
        db[e] = d.sum(0)
        bb[e] = ((b - a + 8) * SUM_ULP * np.abs(d) + 64 * SUM_ULP * np.abs(dy[a:b])).sum(0)
    return (dx, dw, db), (bx, bw, bb)


def check(got, ref, bound, dtype, what=""):
    """|got - ref| <= bound + the rounding of (ref +- bound) to the type."""
    g = f64(got)
    assert g.shape == ref.shape, (what, g.shape, ref.shape)
    lim = bound + HALF_ULP[dtype] * (np.abs(ref) + bound) + 1e-37
    err = np.abs(g - ref)
    bad = ~(err <= lim)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} out of bounds, first at "
                           f"{tuple(np.argwhere(bad)[0])}: got {g[bad][0]}, want {ref[bad][0]}, "
                           f"allowed {lim[bad][0]}")
