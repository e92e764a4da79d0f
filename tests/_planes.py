"""The three-plane form of F32 products restated in numpy, and the relative error
in the norm that tests hold it to."""
import numpy as np

# Relative error of an F32 product, in the norm, for terms of random sign: the
# left-out products of planes take 2^-24 on average; a 64-wide step's sum is
# truncated at each of the 4 accumulations of its large products, half a unit
# of 2^-23 each on average, which is 2^-22; adding the steps, rounded to nearest,
# gives less.  Together below 2^-21; twice that is allowed.  A product of planes
# that is lost costs 1e-5 or more.
F32_NORM = 2.0 ** -20


def planes(x):
    """h + m + l = x, 8 bits each, truncated."""
    def cut(v):
        return (v.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
    h = cut(x)
    m = cut(x - h)
    return h, m, x - h - m


def product(a, b, keep):
    """Sum of the kept products of planes, in 64 bits."""
    p, q = [v.astype(np.float64) for v in planes(a)], [v.astype(np.float64) for v in planes(b)]
    return sum(p[i] @ q[j] for i, j in keep)


SIX = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]
