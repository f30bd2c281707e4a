#!/usr/bin/env python3
"""Fits of the GELU used by the 8-bit product's epilogue (gelu8.cuh).

gelu(x) = max(x, 0) - a T(a), a = |x|, T(a) = 1 - Phi(a) the normal tail.  log2 T
is smooth and nearly quadratic, so T(a) = 2^P(a) with one power of two and a
polynomial of low degree.  A block of negative x has nothing but the tail, and its
scale is its largest value, so what has to be small is the relative error: P
minimises the largest |2^P / T - 1| / (1 + a^2) (linear programming on a grid).
The weight 1 + a^2 is how much a relative error of x itself is magnified in
a T(a), so the bound reads as that of a slightly different x.

`fit()` covers [0, 5.5], `fit_tail()` [5.5, 14], past which a T(a) is below a
thousandth of the smallest code's value at the smallest scale.  Both leading
coefficients are negative: P falls past its range, however large a is.

    python gelu8_fit.py      prints the coefficients and the errors
"""
import numpy as np

DEGREE, TOP = 8, 5.5
TAIL_DEGREE, TAIL_TOP = 5, 14.0


def tail_log2(a):
    from scipy.special import log_ndtr
    return log_ndtr(-a) / np.log(2.0)


def fit(degree=DEGREE, low=0.0, top=TOP, n=4000):
    from scipy.optimize import linprog
    a = low + (top - low) * (1.0 - np.cos(np.pi * np.arange(n) / (n - 1))) / 2.0
    want = tail_log2(a)
    w = np.log(2.0) / (1.0 + a * a) * 1e6
    v = np.polynomial.chebyshev.chebvander((2.0 * a - low - top) / (top - low), degree) * w[:, None]
    one = np.ones((n, 1))
    r = linprog(np.r_[np.zeros(degree + 1), 1.0], A_ub=np.vstack([np.hstack([v, -one]), np.hstack([-v, -one])]),
                b_ub=np.r_[want * w, -want * w], bounds=[(None, None)] * (degree + 1) + [(0, None)], method="highs")
    p = np.polynomial.chebyshev.Chebyshev(r.x[:-1], domain=[low, top]).convert(kind=np.polynomial.Polynomial)
    return p.coef


def fit_tail():
    return fit(TAIL_DEGREE, TOP, TAIL_TOP)


if __name__ == "__main__":
    for c, low, top in ((fit(), 0.0, TOP), (fit_tail(), TOP, TAIL_TOP)):
        a = np.linspace(low, top, 200001)
        err = np.abs(2.0 ** (np.polynomial.polynomial.polyval(a, c) - tail_log2(a)) - 1.0) / (1.0 + a * a)
        print("[%g, %g], constant first:" % (low, top), ", ".join("%.9ef" % x for x in c))
        print("  largest |2^P / T - 1| / (1 + a^2): %.3g" % err.max())
