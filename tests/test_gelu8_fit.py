"""The GELU fit of the 8-bit product's epilogue, on the CPU: the coefficients in the
kernel's header are the fit's, and evaluated in fp32 the way the kernel does
(Horner steps, one rounding each; exp2 within 2^-22) the GELU stays within
2^-20 |x| of x Phi(x)."""
import importlib.util
import re
from pathlib import Path

import numpy as np
from scipy.special import erfc

CSRC = Path(__file__).resolve().parent.parent / "logic-bs-roformer-rs_b200" / "csrc"


def header_coefficients():
    """From the header, highest power of n = -|x| first."""
    text = (CSRC / "gelu8.cuh").read_text()
    body = text[text.index("__device__ __forceinline__ float2 gelu8"):]
    pairs = re.findall(r"f2\((-?\d\.\d+e[+-]\d+)f, (-?\d\.\d+e[+-]\d+)f\)", body)
    assert all(a == b for a, b in pairs)
    return [float(a) for a, _ in pairs]


def test_coefficients_are_the_fit():
    spec = importlib.util.spec_from_file_location("gelu8_fit", CSRC / "gelu8_fit.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    c = m.fit()
    signed = [v * (-1) ** k for k, v in enumerate(c)][::-1]
    got = header_coefficients()
    assert len(got) == m.DEGREE + 1
    a = np.linspace(0.0, 6.0, 20001)
    t = 2.0 ** np.polynomial.polynomial.polyval(a, c)
    h = 2.0 ** np.polyval(np.array(got), -a)
    assert np.abs(t - h).max() < 2e-8  # the printed digits
    np.testing.assert_allclose(got, signed, rtol=1e-6)


def test_error_in_fp32():
    x = np.concatenate([np.linspace(-14, 14, 400001), np.logspace(-30, 1, 5001), -np.logspace(-30, 1, 5001),
                        [-1e4, 1e4, -3e38, 3e38, 0.0]]).astype(np.float32)
    n = -np.abs(x)
    f32 = np.float32
    with np.errstate(over="ignore", invalid="ignore"):
        p = None
        for c in header_coefficients():  # fma: exact product and sum in 64 bits, one rounding
            p = np.full_like(n, f32(c)) if p is None else (p.astype(np.float64) * n + f32(c)).astype(f32)
        t = np.exp2(p.astype(np.float64))
        for worst in (1 - 2.0 ** -22, 1 + 2.0 ** -22):
            g = n.astype(np.float64) * (t * worst).astype(f32) + np.maximum(x, f32(0))
            want = 0.5 * x.astype(np.float64) * erfc(-x.astype(np.float64) / np.sqrt(2.0))
            assert (np.abs(g - want) <= np.abs(x) * 2.0 ** -20).all()
