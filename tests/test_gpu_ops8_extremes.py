"""The 8-bit operators at the ends of what they take: longest rows, most rows, longest K, every output pitch, wide norms
with many rows, and a first call of the tiled product inside a capture."""
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
MAX_COLS = 65535 * 128
PKG = Path(__file__).resolve().parent.parent / "logic-bs-roformer-rs_b200"


@pytest.fixture(scope="module")
def lb():
    import lbrr
    lbrr.lib()
    return lbrr


def rnd(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale).to(dtype)


def divided(x, br):
    """(code bytes, scales) by torch's fp32 division and conversion."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -cols % 128, 0, -rows % br))
    b = v.view(v.shape[0] // br, br, v.shape[1] // 128, 128)
    s = (b.abs().amax((1, 3)) / torch.full((), 448.0, device=x.device)).clamp(min=2.0 ** -126)
    q = (b / s[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.reshape(v.shape)[:rows, :cols].contiguous().view(torch.uint8), s.t().contiguous()


def values(q, s, br):
    rows, cols = q.shape
    r = torch.arange(rows, device=q.device) // br
    c = torch.arange(cols, device=q.device) // 128
    return q.double() * s.double()[c][:, r].t()


@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("rows,cols", [(3, MAX_COLS), (2, MAX_COLS - 1), ((1 << 24) + 3, 1), (1 << 21, 130)])
def test_quant8_longest(lb, br, rows, cols):
    x = rnd((rows, cols), 1, torch.float16)
    want, ws = divided(x, br)
    q, s = lb.empty8(rows, cols, br)
    lb.quant8(x, q, s, block_rows=br)
    torch.cuda.synchronize()
    assert torch.equal(s, ws) and torch.equal(q.contiguous().view(torch.uint8), want)


@pytest.mark.parametrize("m,n", [(1, 1), (2, 130), (70, 3), (20000, 5)])
def test_gemm8_longest_k(lb, m, n):
    """K up to the limit (fewer rows where memory asks for it): the sums of tens of thousands of blocks."""
    k = MAX_COLS if m < 100 else 40003
    a, sa = lb.empty8(m, k)
    w, sw = lb.empty8(n, k, 128)
    lb.quant8(rnd((m, k), 1, torch.float16), a, sa)
    lb.quant8(rnd((n, k), 2, torch.float16, 0.02), w, sw, block_rows=128)
    out = torch.zeros(m, n, device="cuda")
    lb.gemm8(a, sa, w, sw, out)
    lb.op_sync()
    want, size = torch.zeros(m, n, dtype=torch.float64, device="cuda"), torch.zeros(m, n, dtype=torch.float64, device="cuda")
    step = 128 * 4096 if m < 100 else 128 * 64
    for at in range(0, k, step):
        b = slice(at // 128, (min(at + step, k) + 127) // 128)
        a64, w64 = values(a[:, at:at + step], sa[b], 1), values(w[:, at:at + step], sw[b], 128)
        want += a64 @ w64.t()
        size += a64.abs() @ w64.abs().t()
    blocks = -(-k // 128)
    assert ((out.double() - want).abs() <= (128 + 2 * blocks + 8) * 2 * U * size).all()


@pytest.mark.parametrize("m,n", [((1 << 22) + 7, 1), (130, 65536), (1, 1 << 20)])
def test_gemm8_most_rows_and_columns(lb, m, n):
    k = 40
    a, sa = lb.empty8(m, k)
    w, sw = lb.empty8(n, k, 128)
    lb.quant8(rnd((m, k), 1), a, sa)
    lb.quant8(rnd((n, k), 2), w, sw, block_rows=128)
    out = torch.zeros(m, n, device="cuda")
    lb.gemm8(a, sa, w, sw, out)
    lb.op_sync()
    a64, w64 = values(a, sa, 1), values(w, sw, 128)
    for at in range(0, m, 1 << 16):
        p = a64[at:at + (1 << 16)]
        want, size = p @ w64.t(), p.abs() @ w64.abs().t()
        assert ((out[at:at + (1 << 16)].double() - want).abs() <= 138 * 2 * U * size).all()


@pytest.mark.parametrize("m,n,k", [(4097, 333, 200), (6000, 129, 70), (300, 333, 200), (33, 70, 300)])
def test_gelu_rows_at_any_offset(lb, m, n, k):
    """The same codes wherever the output's rows start, and nothing beside them is written."""
    a, sa = lb.empty8(m, k)
    w, sw = lb.empty8(n, k, 128)
    lb.quant8(rnd((m, k), 1), a, sa)
    lb.quant8(rnd((n, k), 2, scale=k ** -0.5), w, sw, block_rows=128)
    bias = rnd((n,), 3)
    q0, s0 = lb.empty8(m, n)
    lb.gemm8_gelu_quant8(a, sa, w, sw, bias, q0, s0)
    for shift in (0, 1, 2, 3, 4, 8, 15, 16):
        for pitch in (n, n + 1, n + 2, n + 3, n + -n % 4, n + -n % 16):
            buf = torch.full((m * pitch + shift + 32,), 0x55, dtype=torch.uint8, device="cuda")
            q = buf.view(torch.float8_e4m3fn).as_strided((m, n), (pitch, 1), shift)
            s = torch.full_like(s0, -7.0)
            lb.gemm8_gelu_quant8(a, sa, w, sw, bias, q, s)
            torch.cuda.synchronize()
            codes = buf.as_strided((m, n), (pitch, 1), shift)
            assert torch.equal(codes, q0.view(torch.uint8)) and torch.equal(s, s0), (shift, pitch)
            codes.fill_(0x55)
            assert (buf == 0x55).all()


@pytest.mark.parametrize("xt,rt", [(torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                   (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,cols,pad", [(700, 20000, 0), (301, 16385, 0), (333, 32768, 8), (150, 17003, 5),
                                           (2000, 5000, 3), (5001, 600, 0)])
def test_norm_of_many_wide_rows(lb, xt, rt, rows, cols, pad):
    """Several rows a block, one after the other."""
    x, r = rnd((rows, cols + pad), 1, xt)[:, :cols], rnd((rows, cols + pad), 2, rt)[:, :cols]
    gamma = 1.0 + 0.1 * rnd((cols,), 3)
    y = torch.empty(rows, cols, dtype=rt, device="cuda")
    q, s = lb.empty8(rows, cols)
    lb.add_norm_quant8(x, r, gamma, y, q, s, eps=1.0)
    torch.cuda.synchronize()
    assert torch.equal(y, (x.float() + r.float()).to(rt))
    v = x.double() + r.double()
    n = v / (v.pow(2).mean(1, keepdim=True) + 1.0).sqrt() * gamma.double()
    top = torch.nn.functional.pad(n, (0, -cols % 128)).view(rows, -1, 128).abs().amax(2).t() / 448.0
    # the norm is within 2^-18 of itself (the bound of the norm's tests); codes are rounded by half a step
    assert ((s.double() - top).abs() <= top * (2.0 ** -18 + 2 * U)).all()
    u = n / s.double().repeat_interleave(128, 0)[:cols].t()
    step = torch.maximum(u.abs() * 2.0 ** -4, torch.full_like(u, 2.0 ** -10))
    assert ((q.double() - u).abs() <= step + u.abs() * (2.0 ** -18 * (1 + 2.0 ** -4) + 2.0 ** -21)).all()


FIRST_TILED = """
import sys
sys.path.insert(0, sys.argv[1])
import torch, lbrr
def operands(m, n, k):
    a, sa = lbrr.empty8(m, k); w, sw = lbrr.empty8(n, k, 128)
    lbrr.quant8(torch.ones(m, k, device="cuda"), a, sa); lbrr.quant8(torch.ones(n, k, device="cuda"), w, sw, 128)
    return a, sa, w, sw
out = torch.zeros(4, 128, device="cuda")
lbrr.gemm8(*operands(4, 128, 128), out)  # the split product: the status word exists now
big, res = operands(9000, 200, 300), torch.zeros(9000, 200, device="cuda")
q, s = lbrr.empty8(9000, 200)
st = torch.cuda.Stream()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=st):
    lbrr.gemm8(*big, res, stream=torch.cuda.current_stream())
    lbrr.gemm8_gelu_quant8(*big, None, q, s, stream=torch.cuda.current_stream())
assert (res == 0).all()
g.replay(); torch.cuda.synchronize(); lbrr.op_sync()
assert (res - 300.0).abs().max() < 1e-3 and (s * 448 - 300.0).abs().max() < 1e-3 and (q.float() == 448.0).all()
print("ok")
"""


def test_first_tiled_product_inside_a_capture(tmp_path):
    script = tmp_path / "first_tiled.py"
    script.write_text(FIRST_TILED)
    r = subprocess.run([sys.executable, str(script), str(PKG)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("m,n,k", [(62, 1024, 256), (9000, 260, 256)])
def test_infinite_sums_spoil_their_block_only(lb, m, n, k):
    """A bias of -infinity: gelu is not a number there, and the block with it; without GELU the sum is -infinity."""
    a, sa = lb.empty8(m, k)
    w, sw = lb.empty8(n, k, 128)
    lb.quant8(rnd((m, k), 1), a, sa)
    lb.quant8(rnd((n, k), 2, scale=k ** -0.5), w, sw, block_rows=128)
    bias = rnd((n,), 3)
    q0, s0 = lb.empty8(m, n)
    lb.gemm8_gelu_quant8(a, sa, w, sw, bias, q0, s0)
    bias[130] = -math.inf
    q, s = lb.empty8(m, n)
    lb.gemm8_gelu_quant8(a, sa, w, sw, bias, q, s)
    out = torch.empty(m, n, device="cuda")
    lb.gemm8(a, sa, w, sw, out, bias=bias)
    lb.op_sync()
    other = torch.arange(n, device="cuda") // 128 != 1
    assert torch.isnan(s[1]).all() and torch.isnan(q[:, ~other].float()).all()
    assert torch.equal(s[torch.arange(s.shape[0]) != 1], s0[torch.arange(s.shape[0]) != 1])
    assert torch.equal(q.view(torch.uint8)[:, other], q0.view(torch.uint8)[:, other])
    assert (out[:, 130] == -math.inf).all() and torch.isfinite(out[:, torch.arange(n, device="cuda") != 130]).all()
