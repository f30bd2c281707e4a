"""The codes of quant8 are those of the fp32 quotient v / scale, rounded to nearest even: bit for bit what a
division and a conversion give.  The scale is max|v| / 448, rounded once, so both outputs have one right answer."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def lb():
    import lbrr
    lbrr.lib()
    return lbrr


def divided(x, br):
    """(code bytes, scales) by torch's fp32 division and conversion."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -cols % 128, 0, -rows % br))
    b = v.view(v.shape[0] // br, br, v.shape[1] // 128, 128)
    # torch divides by a number as a product with its reciprocal; by a tensor it divides
    s = (b.abs().amax((1, 3)) / torch.full((), 448.0, device=x.device)).clamp(min=2.0 ** -126)
    q = (b / s[:, None, :, None]).to(torch.float8_e4m3fn)
    q = q.reshape(v.shape)[:rows, :cols].contiguous().view(torch.uint8)
    return q, s.t().contiguous()


def same(lb, x, br):
    want, ws = divided(x, br)
    q, s = lb.empty8(*x.shape, br)
    lb.quant8(x, q, s, block_rows=br)
    torch.cuda.synchronize()
    assert torch.equal(s, ws)
    got = q.contiguous().view(torch.uint8)
    assert torch.equal(got, want), int((got != want).sum())


def values(rows, cols, seed, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(
        0.7 * torch.randn(cols, generator=g, device="cuda"))).to(dtype)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (62, 256), (5000, 512), (40000, 64), (4000, 588), (3001, 257), (129, 5000)])
def test_codes(lb, kind, br, rows, cols):
    same(lb, values(rows, cols, rows + cols, TYPES[kind]), br)


@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("power", [-149, -140, -130, -120, -100, -62, -60, -58, -20, 60, 118, 125])
def test_codes_at_every_size(lb, br, power):
    """Scales from the smallest to the largest, the remainders of the division below the normal range among them."""
    x = values(640, 512, 7, torch.float32)
    x = (x / x.abs().max()).double() * 2.0 ** power
    same(lb, x.float(), br)


def test_every_half_over_many_tops(lb):
    """Every finite fp16 value up to the block's largest, for many largest values."""
    h = torch.arange(0x7C00, dtype=torch.int32, device="cuda").to(torch.int16).view(torch.float16)
    g = torch.Generator(device="cuda").manual_seed(1)
    for top in (0x3C00, 0x3C01, 0x3BFF, 0x5555, 0x7BFF, 0x0400, 0x0001, 0x2E66, 0x4248):
        row = h[:top + 1]
        n = row.numel() // 127 * 127 + 127
        row = torch.nn.functional.pad(row, (0, n - row.numel())).view(-1, 127)
        row = torch.cat([row, h[top].expand(row.shape[0], 1)], 1)
        flip = torch.randint(0, 2, row.shape, generator=g, device="cuda").half() * 2 - 1
        same(lb, row * flip, 1)


def test_zeros_keep_their_sign(lb):
    x = torch.zeros(4, 256, device="cuda")
    x[0, 3], x[1, 0], x[1, 1], x[2, 200] = -0.0, -0.0, 5.0, -1e-38
    same(lb, x, 1)
    same(lb, x, 128)
    q, s = lb.empty8(4, 256)
    lb.quant8(x, q, s)
    assert math.copysign(1.0, float(q[0, 3].float())) == -1.0


def test_bad_blocks_hold_the_same_nan(lb):
    x = values(8, 512, 3, torch.float32)
    x[2, 140], x[5, 1] = math.inf, math.nan
    q, s = lb.empty8(8, 512)
    lb.quant8(x, q, s)
    torch.cuda.synchronize()
    codes = q.view(torch.uint8)
    assert torch.isnan(s[1, 2]) and torch.isnan(s[0, 5]) and int(torch.isnan(s).sum()) == 2
    assert (codes[2, 128:256] == 0x7F).all() and (codes[5, :128] == 0x7F).all()
