"""The three-plane form of F32 products, restated in numpy: what the planes
hold, what the six products leave out, and that a form which lost a plane or a
product would not pass the norm bound the GPU tests use."""
import numpy as np
import pytest

from _planes import F32_NORM, SIX, planes, product


def test_planes_hold_every_value():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal(1 << 16) * 2.0 ** rng.integers(-80, 100, 1 << 16)).astype(np.float32)
    h, m, l = planes(x)
    assert np.array_equal(h.astype(np.float64) + m + l, x.astype(np.float64))
    for v in (h, m, l):
        assert not (v.view(np.uint32) & 0xFFFF).any()            # each is a bf16 value
        assert (v * np.sign(x) >= 0).all()                       # of x's sign


def test_what_the_six_products_leave_out():
    """m l + l m + l l: up to 2^-21 of a term (7.8 units of 2^-24 here), 0.7 units
    of 2^-24 on average, toward zero."""
    rng = np.random.default_rng(2)
    x = np.concatenate([rng.standard_normal(1 << 18), [np.uint32(0x3F80FFFF).view(np.float32)] * 2]).astype(np.float32)
    y = np.concatenate([rng.standard_normal(1 << 18), [np.uint32(0x3F80FFFF).view(np.float32)] * 2]).astype(np.float32)
    p, q = [v.astype(np.float64) for v in planes(x)], [v.astype(np.float64) for v in planes(y)]
    lost = 1 - sum(p[i] * q[j] for i, j in SIX) / (x.astype(np.float64) * y)
    assert (lost >= -1e-15).all() and lost.max() < 2.0 ** -20.9
    assert lost.max() > 2.0 ** -22 and 0.5 < lost.mean() * 2 ** 24 < 1.0


@pytest.mark.parametrize("K", [192, 640, 1536])
def test_norm_bound_sees_a_lost_plane(K):
    rng = np.random.default_rng(K)
    a, b = rng.standard_normal((40, K)).astype(np.float32), rng.standard_normal((K, 50)).astype(np.float32)
    ref = a.astype(np.float64) @ b

    def off(keep):
        return np.linalg.norm(product(a, b, keep) - ref) / np.linalg.norm(ref)

    assert off(SIX) <= 2.0 ** -23
    for i, j in SIX:
        assert off([k for k in SIX if k != (i, j)]) > 4 * F32_NORM, (i, j)
    swapped = [(2, 1) if k == (2, 0) else k for k in SIX]        # a plane paired wrongly
    assert off(swapped) > 4 * F32_NORM
