"""gemm8_gelu_quant8 on blocks whose values are all negative: their scale is a value of the normal tail, so the error
is bounded relative to max |gelu| of the block.

Bounds: h = A W^T + bias is within tol (the bound of the product's tests, repeated here), and gelu within
2^-19 (1 + h^2) of itself for h < 0, 2^-19 |h| for h >= 0 (the epilogue's fits and their roundings), and within 1e-10
for h below -5.5 beside an h of 0.3 or more, where that is a 2^-11 of half a step of the smallest code.  An h that is
off by tol moves gelu by the difference at h - tol and h + tol, gelu being monotone but around its minimum at -0.75,
where that difference misses at most 1.13 tol^2 / 2."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def lb():
    import lbrr
    lbrr.lib()
    return lbrr


def expand(s, rows, cols, br):
    r = torch.arange(rows, device=s.device) // br
    c = torch.arange(cols, device=s.device) // 128
    return s[c][:, r].t()


def tops(v):
    v = torch.nn.functional.pad(v, (0, -v.shape[1] % 128))
    return v.abs().view(v.shape[0], -1, 128).amax(2).t()


def gelu(h):
    return 0.5 * h * torch.special.erfc(-h / math.sqrt(2.0))


def check(lb, m, n, k, bias, spread, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda")
    w = torch.randn(n, k, generator=g, device="cuda") * (spread / math.sqrt(k))
    a, sa = lb.empty8(m, k)
    b, sb = lb.empty8(n, k, 128)
    lb.quant8(x, a, sa)
    lb.quant8(w, b, sb, block_rows=128)
    a64, b64 = a.double() * expand(sa.double(), m, k, 1), b.double() * expand(sb.double(), n, k, 128)
    blocks = -(-k // 128)
    h = a64 @ b64.t() + bias.double()
    tol = (128 + 2 * blocks + 8) * 2 * U * (a64.abs() @ b64.abs().t()) + blocks * U * bias.double().abs()
    tol = tol + U * (h.abs() + tol)
    want = gelu(h)
    moved = torch.maximum((gelu(h - tol) - want).abs(), (gelu(h + tol) - want).abs()) + 0.6 * tol * tol
    lim = moved + torch.where(h < 0, want.abs() * (1 + h * h), h.abs()) * 2.0 ** -19 + 2.0 ** -149
    high = torch.nn.functional.pad(h + tol, (0, -n % 128), value=-math.inf).view(m, -1, 128).amax(2)
    lim = lim + torch.where((h < -5.5) & (high.repeat_interleave(128, 1)[:, :n] >= 0.3), 1e-10, 0.0)
    q, s = lb.empty8(m, n)
    lb.gemm8_gelu_quant8(a, sa, b, sb, bias, q, s)
    lb.op_sync()
    s64, scale = s.double(), (tops(want) / 448.0).clamp(min=2.0 ** -126)
    bound = tops(lim) / 448.0 + scale * 2 * U
    err = (s64 - scale).abs()
    assert (err <= bound).all(), float((err / bound).max())
    # the codes: half a step of e4m3 (2^-10 below the normal range) for the value's error over the block's own scale
    e = expand(s64, m, n, 1)
    u = want / e
    step = torch.maximum(u.abs() * 2.0 ** -4, torch.full_like(u, 2.0 ** -10))
    off = (q.double() - u).abs() - step - lim / e * (1 + 2.0 ** -4) - u.abs() * 2.0 ** -21
    assert (off <= 0).all(), float(off.max())
    return h, (err / scale).max().item()


SHAPES = [(1, 128, 128), (62, 1024, 256), (33, 129, 250), (5, 1, 40), (700, 257, 300),  # split
          (9000, 129, 256), (12000, 257, 128), (4097, 1024, 256)]                        # tiled


@pytest.mark.parametrize("shift", [-0.5, -2.0, -4.0, -4.9, -5.1, -5.4, -5.6, -7.0, -10.0, -12.5, -13.4, -20.0, 3.0])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_shifted_blocks(lb, m, n, k, shift):
    """Every value near `shift`: whole blocks in the tail, and a last block of one column."""
    bias = torch.full((n,), shift, device="cuda")
    check(lb, m, n, k, bias, 0.1)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_mixed_blocks(lb, m, n, k):
    """Blocks on both sides of the fits' border, spread values, and columns far out beside ordinary ones."""
    g = torch.Generator(device="cuda").manual_seed(n)
    bias = 3.0 * torch.randn(n, generator=g, device="cuda") - 3.0
    check(lb, m, n, k, bias, 1.0)
    bias[::7] = -9.0
    bias[3::11] = 40.0
    check(lb, m, n, k, bias, 2.0, seed=2)


@pytest.mark.parametrize("m,n,k", [(62, 1024, 256), (4097, 1024, 256)])
def test_a_rows_result_does_not_depend_on_the_others(lb, m, n, k):
    """Rows in the tail beside ordinary ones change nothing in those."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(m, k, generator=g, device="cuda")
    w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
    b, sb = lb.empty8(n, k, 128)
    lb.quant8(w, b, sb, block_rows=128)
    bias = torch.zeros(n, device="cuda")

    def out(x):
        a, sa = lb.empty8(m, k)
        lb.quant8(x, a, sa)
        q, s = lb.empty8(m, n)
        lb.gemm8_gelu_quant8(a, sa, b, sb, bias, q, s)
        lb.op_sync()
        return q.contiguous().view(torch.uint8), s

    q0, s0 = out(x)
    loud = x.clone()
    loud[::5] *= 20.0
    q1, s1 = out(loud)
    keep = torch.arange(m, device="cuda") % 5 != 0
    assert torch.equal(q0[keep], q1[keep]) and torch.equal(s0[:, keep], s1[:, keep])
