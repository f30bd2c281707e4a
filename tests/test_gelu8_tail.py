"""The GELU of the 8-bit product's epilogue on negative x, on the CPU: relative to gelu(x) itself, which is all that
a block of negative values and its scale hold.

Both fits keep 2^P within 2^-20 (1 + a^2) of the normal tail, a = |x|.  In fp32, P is a chain of FMAs whose last
results are near |P| and whose coefficients are rounded: three roundings of |P| at most, 3 x 2^-24 |P| ln 2 relative,
and |P| <= 1 + 1.2 a + 0.73 a^2 (the tail's logarithm) is below 3 (1 + a^2), so below 2^-21 (1 + a^2); exp2 within
2^-22 and the product's 2^-24 join them.  Together below 2^-19 (1 + a^2), and 2^-149 for results below the normal range."""
import importlib.util
import re
from pathlib import Path

import numpy as np
import pytest
from scipy.special import log_ndtr

CSRC = Path(__file__).resolve().parent.parent / "logic-bs-roformer-rs_b200" / "csrc"
f32 = np.float32


def fits():
    spec = importlib.util.spec_from_file_location("gelu8_fit", CSRC / "gelu8_fit.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def coefficients(function):
    """Those of a function of the header, highest power of n = -|x| first; the added exponent apart."""
    text = (CSRC / "gelu8.cuh").read_text()
    body = text[text.index("__device__ __forceinline__ float2 %s(" % function):]
    body = body[:body.index("\n}\n")]
    up = 32.0 if "32.0f - " in body else 0.0
    pairs = re.findall(r"f2\((?:32\.0f )?(-? ?\d\.\d+e[+-]\d+)f, (?:32\.0f )?(-? ?\d\.\d+e[+-]\d+)f\)", body)
    assert all(a == b for a, b in pairs)
    return [float(a.replace(" ", "")) for a, _ in pairs], up


def horner(c, up, n):
    p = np.full_like(n, f32(c[0]))
    for k, v in enumerate(c[1:], 2):
        v = f32(v + up) if k == len(c) else f32(v)
        p = (p.astype(np.float64) * n + v).astype(f32)  # fma: exact product and sum in 64 bits, one rounding
    return p


def gelu(x, worst):
    """The kernel's steps for x <= 0, exp2 off by the factor `worst`."""
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        main, up = coefficients("gelu8")
        t = (np.exp2(horner(main, up, x).astype(np.float64)) * worst).astype(f32)
        return (x.astype(np.float64) * t).astype(f32)


def before(x, worst):
    """What the kernel gives its GELU instead of x <= -5.5."""
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        tail, up = coefficients("before_gelu8")
        p = horner(tail, up, x)
        t = (np.exp2(p.astype(np.float64)) * worst).astype(f32)
        t[p < -126] = 0.0  # .ftz
        y = ((x * f32(2.0 ** (1 - up))).astype(np.float64) * t).astype(f32)
        return np.where(x < -5.5, y, x)


@pytest.mark.parametrize("worst", [1 - 2.0 ** -22, 1 + 2.0 ** -22])
def test_relative_error(worst):
    x = -np.concatenate([np.linspace(0, 14, 700001), np.logspace(-30, 1, 20001)]).astype(f32)
    x = x[x >= -14.0]
    a = x.astype(np.float64)
    want = a * np.exp(log_ndtr(a))
    err = np.abs(gelu(before(x, worst), worst).astype(np.float64) - want)
    lim = np.abs(want) * 2.0 ** -19 * (1 + a * a) + 2.0 ** -149
    assert (err <= lim).all(), (x[err > lim][:5], (err / np.abs(want))[err > lim][:5])


def test_past_the_fits_the_tail_vanishes():
    x = -np.concatenate([np.linspace(14, 60, 20001), np.logspace(1.8, 38.5, 4001)]).astype(f32)
    g = gelu(before(x, 1.0), 1.0)
    # a T(a) falls from 1.1e-43 at 14; the smallest code that is not zero stands for 2^-126 x 2^-9 = 2.3e-41
    assert (np.abs(g) <= 2e-43).all() and not np.isnan(g).any()


def test_tail_coefficients_are_the_fit():
    m = fits()
    c = m.fit_tail()
    got, up = coefficients("before_gelu8")
    assert len(got) == m.TAIL_DEGREE + 1 and up == 32.0
    np.testing.assert_allclose(got, [v * (-1) ** k for k, v in enumerate(c)][::-1], rtol=1e-6)


def test_the_fits_themselves():
    m = fits()
    for c, low, top in ((m.fit(), 0.0, m.TOP), (m.fit_tail(), m.TOP, m.TAIL_TOP)):
        a = np.linspace(low, top, 100001)
        p = np.polynomial.polynomial.polyval(a, c)
        assert (np.abs(np.exp2(p - log_ndtr(-a) / np.log(2.0)) - 1) <= 2.0 ** -20 * (1 + a * a)).all()
        assert c[-1] < 0.0
