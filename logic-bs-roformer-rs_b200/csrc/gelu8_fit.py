#!/usr/bin/env python3
"""Fit of the GELU used by the 8-bit product's epilogue (gelu8.cuh).

gelu(x) = max(x, 0) - a T(a), a = |x|, T(a) = 1 - Phi(a) the normal tail.  log2 T
is smooth and nearly quadratic, so T(a) = 2^P(a) with one power of two and a
polynomial of low degree.  P minimises the largest |2^P - T| on [0, 6] (linear
programming on a grid; the weight T ln 2 turns an error of P into one of T); past
6, T < 1e-9 and P keeps falling (its leading coefficient is negative), so T only
has to vanish there.  The error of gelu is a times that of T.

    python gelu8_fit.py      prints the coefficients and the error
"""
import numpy as np

DEGREE, TOP = 5, 6.0


def tail_log2(a):
    from scipy.special import log_ndtr
    return log_ndtr(-a) / np.log(2.0)


def fit(degree=DEGREE, top=TOP, n=4000):
    from scipy.optimize import linprog
    a = np.linspace(0.0, top, n)
    want = tail_log2(a)
    w = 2.0 ** want * np.log(2.0) * 1e3
    v = np.polynomial.chebyshev.chebvander(2.0 * a / top - 1.0, degree) * w[:, None]
    one = np.ones((n, 1)) * 1e3
    r = linprog(np.r_[np.zeros(degree + 1), 1.0], A_ub=np.vstack([np.hstack([v, -one]), np.hstack([-v, -one])]),
                b_ub=np.r_[want * w, -want * w], bounds=[(None, None)] * (degree + 1) + [(0, None)], method="highs")
    p = np.polynomial.chebyshev.Chebyshev(r.x[:-1], domain=[0.0, top]).convert(kind=np.polynomial.Polynomial)
    return p.coef


if __name__ == "__main__":
    c = fit()
    a = np.linspace(0.0, 14.0, 200001)
    err = np.abs(2.0 ** np.polynomial.polynomial.polyval(a, c) - 2.0 ** tail_log2(a)).max()
    print("coefficients, constant first:", ", ".join("%.9ef" % x for x in c))
    print("largest |2^P - T| on [0, 14]: %.3g" % err)
