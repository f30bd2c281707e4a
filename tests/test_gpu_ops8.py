"""8-bit operators on the GPU against their definitions in 64 bits.

Bounds, derived from the arithmetic (u = 2^-24, half an ulp of fp32):

* e4m3 rounds by at most half a step: 2^-4 of the value, or 2^-10 below the
  smallest normal (2^-6); the code is of v * (1/s), two fp32 roundings more.
* A norm's sum of squares: at most 32 terms per lane in sequence, 5 shuffle
  steps, at most 32 partial sums: 70 u, halved by the root; the sum y, the mean,
  the root, the division and two products add under 8 u.  Together below 2^-18.
* A product's block sum: products of e4m3 values are exact in fp32; 128 adds,
  each within 2u (an adder that truncates) of the sum of magnitudes; the product
  of the two scales, the scaling and the running total add 4u per block.  So
  |error| <= (128 + 2 * blocks + 8) * 2u * S with S = sum |a||w| in true values.
  The running total starts from the bias: its magnitude joins every addition's,
  so blocks * u * |bias| more.
* gelu' is at most 1.13; the erf itself is within 2^-20.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def lb():
    import lbrr
    lbrr.lib()
    return lbrr


def rnd(shape, seed, dtype=torch.float32, scale=1.0, pad=0, shift=0):
    """Seeded normals; pad/shift: a view whose rows are `pad` longer and start `shift` in."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randn(shape[0], shape[1] + pad, generator=g, device="cuda") * scale
    t = t.to(dtype)
    return t[:, shift:shift + shape[1]]


def out8(rows, cols, br=1, pitch=None, code=0x55):
    """(q, scales, whole q buffer) with canary bytes."""
    pitch = pitch or cols + -cols % 16
    buf = torch.full((rows + 1, pitch), code, dtype=torch.uint8, device="cuda")
    q = buf.view(torch.float8_e4m3fn)[:rows, :cols]
    s = torch.full((-(-cols // 128), -(-rows // br)), -7.0, device="cuda")
    return q, s, buf


def canary_kept(buf, rows, cols, code=0x55):
    return bool((buf[:rows, cols:] == code).all()) and bool((buf[rows] == code).all())


def expand(s, rows, cols, br):
    r = torch.arange(rows, device=s.device) // br
    c = torch.arange(cols, device=s.device) // 128
    return s[c][:, r].t()


def true_scales(v, br):
    rows, cols = v.shape
    v = torch.nn.functional.pad(v, (0, -cols % 128, 0, -rows % br))
    top = v.abs().view(v.shape[0] // br, br, -1, 128).amax((1, 3))
    return (top / 448.0).clamp(min=2.0 ** -126).t()


def check8(q, s, v, br, tol_v, tol_s):
    """q, s hold v (64-bit) whose own error is tol_v (absolute, per value); tol_s: of the scales (relative)."""
    rows, cols = v.shape
    s64 = s.double()
    assert ((s64 - true_scales(v, br)).abs() <= tol_s * true_scales(v, br)).all()
    e = expand(s64, rows, cols, br)
    got = q.double()
    u = v / e
    step = torch.maximum(u.abs() * 2.0 ** -4, torch.full_like(u, 2.0 ** -10))
    err = (got - u).abs()
    lim = step + (tol_v / e) * (1 + 2.0 ** -4) + u.abs() * 2.0 ** -21
    assert (err <= lim).all(), float((err - lim).max())


# ---- quant8 ------------------------------------------------------------------
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("rows,cols,pad,shift", [
    (1, 1, 0, 0), (1, 128, 0, 0), (1, 129, 0, 0), (3, 127, 0, 0), (127, 256, 0, 0), (128, 128, 8, 8), (129, 257, 3, 1),
    (33, 300, 4, 0), (62, 255, 1, 1), (1000, 777, 23, 16), (5, 8192, 0, 0), (2294, 512, 0, 0), (1024, 256, 0, 0)])
def test_quant8(lb, kind, br, rows, cols, pad, shift):
    x = rnd((rows, cols), rows * 1000 + cols, TYPES[kind], 3.0, pad, shift)
    q, s, buf = out8(rows, cols, br)
    lb.quant8(x, q, s, block_rows=br)
    torch.cuda.synchronize()
    v = x.double()
    check8(q, s, v, br, torch.zeros_like(v), U)  # x is exact; top / 448 is rounded once
    assert canary_kept(buf, rows, cols)


def in_nan(x, pitch, shift):
    """x as a view of a buffer of NaN: rows `pitch` apart, the first `shift` values in."""
    buf = torch.full((x.shape[0] * pitch + shift + x.shape[1],), math.nan, dtype=x.dtype, device="cuda")
    view = buf.as_strided(x.shape, (pitch, 1), shift)
    view.copy_(x)
    return view


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("rows,cols", [(5, 1), (9, 8), (70, 100), (131, 127), (33, 129), (40, 249), (64, 255), (300, 256),
                                       (37, 263), (129, 600)])
def test_quant8_rows_at_any_offset(lb, kind, br, rows, cols):
    """The same bits wherever rows start; what stands around them is neither read as theirs nor written."""
    x = rnd((rows, cols), 31 * rows + cols, TYPES[kind])
    q0, s0, _ = out8(rows, cols, br)
    lb.quant8(x.contiguous() if cols % 8 == 0 else in_nan(x, cols + -cols % 8, 0), q0, s0, block_rows=br)
    for shift in range(8):
        for pitch in (cols, cols + 1, cols + 3 + -cols % 8):
            q, s, buf = out8(rows, cols, br, pitch=cols + shift)
            lb.quant8(in_nan(x, pitch, shift), q, s, block_rows=br)
            torch.cuda.synchronize()
            assert torch.equal(q.view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s, s0), (shift, pitch)
            assert canary_kept(buf, rows, cols)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("br", [1, 128])
def test_quant8_special_values(lb, kind, br):
    dt = TYPES[kind]
    x = torch.zeros(256, 512, dtype=dt, device="cuda")
    x[0, 5], x[0, 6], x[0, 7] = -0.0, 1.0, -2.0 ** -14
    x[1, 130] = math.inf
    x[1, 131] = 3.0
    x[128, 300] = math.nan
    x[129, 301] = -math.inf
    x[200, 511] = torch.finfo(dt).max
    x[201, 510] = torch.finfo(dt).tiny
    q, s, _ = out8(256, 512, br)
    lb.quant8(x, q, s, block_rows=br)
    torch.cuda.synchronize()
    bad = torch.zeros(4, 256 // br, dtype=torch.bool, device="cuda")
    bad[1, 1 // br] = bad[2, 128 // br] = bad[2, 129 // br] = True
    assert torch.equal(torch.isnan(s), bad)
    assert torch.equal(torch.isnan(q.float()), expand(bad, 256, 512, br))
    v = torch.where(expand(bad, 256, 512, br), torch.zeros((), dtype=torch.float64, device="cuda"), x.double())
    ok = torch.where(torch.isnan(q.float()), torch.zeros((), device="cuda"), q.float())
    s0 = torch.where(bad, torch.full_like(s, 2.0 ** -126), s)
    check8(ok, s0, v, br, torch.zeros_like(v), U)
    empty = (x == 0).all(1)
    if br == 1:
        assert (q[empty].float() == 0).all() and (s[:, empty] == 2.0 ** -126).all()
        assert q[201, 510].item() == 448.0 or kind != "f16"


def test_quant8_rows_far_apart(lb):
    """Offsets past 2^31 elements on both sides."""
    rows, cols, ld = 1100, 200, 2 ** 21
    big = torch.zeros(rows, ld, dtype=torch.float16, device="cuda")
    big[:, 7 * 8:7 * 8 + cols] = rnd((rows, cols), 5, torch.float16)
    x = big[:, 56:56 + cols]
    qb = torch.zeros(rows, ld, dtype=torch.uint8, device="cuda")
    q = qb.view(torch.float8_e4m3fn)[:, 32:32 + cols]
    s = torch.zeros(2, rows, device="cuda")
    assert (rows - 1) * ld > 2 ** 31
    lb.quant8(x, q, s)
    torch.cuda.synchronize()
    v = x.double()
    check8(q, s, v, 1, torch.zeros_like(v), U)
    assert int((qb != 0).sum()) == int((qb[:, 32:32 + cols] != 0).sum())


# ---- add_norm_quant8 -----------------------------------------------------------
def true_norm(y, gamma, eps):
    d = y.shape[1]
    rms = ((y * y).mean(1, keepdim=True) + eps).sqrt().clamp(min=1e-12 / math.sqrt(d))
    return y / rms * gamma.double()


def check_norm(q, s, n):
    check8(q, s, n, 1, n.abs() * 2.0 ** -18, 2.0 ** -18)


@pytest.mark.parametrize("xt,rt", [("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("rows,cols,pad,shift", [
    (1, 1, 0, 0), (2, 7, 0, 0), (1, 128, 0, 0), (5, 129, 0, 0), (62, 256, 0, 0), (63, 257, 0, 0), (9, 384, 8, 8),
    (100, 513, 3, 1), (17, 1000, 0, 0), (4, 1024, 0, 0), (4, 1025, 7, 0), (3, 5000, 0, 0), (3, 8192, 8, 0),
    (2, 8193, 0, 0), (2, 16384, 0, 0), (2, 32768, 0, 0)])
def test_add_norm_quant8(lb, xt, rt, rows, cols, pad, shift):
    x = rnd((rows, cols), cols, TYPES[xt], 0.5, pad, shift)
    r = rnd((rows, cols), cols + 1, TYPES[rt], 2.0, pad, shift)
    gamma = 1.0 + 0.2 * rnd((1, cols), 3)[0]
    y = torch.full((rows + 1, cols + pad), 9.0, dtype=TYPES[rt], device="cuda")
    yv = y[:rows, shift:shift + cols]
    q, s, buf = out8(rows, cols)
    lb.add_norm_quant8(x, r, gamma, yv, q, s, eps=1e-6)
    torch.cuda.synchronize()
    y64 = x.double() + r.double()
    assert torch.equal(yv, (x.float() + r.float()).to(TYPES[rt]))  # one fp32 sum, rounded once
    check_norm(q, s, true_norm(y64, gamma, 1e-6))
    assert canary_kept(buf, rows, cols) and (y[rows] == 9.0).all()
    if pad:
        assert (y[:rows, shift + cols:] == 9.0).all() and (y[:rows, :shift] == 9.0).all()
    # without storing the sum, and the norm of x alone
    q2, s2, _ = out8(rows, cols)
    lb.add_norm_quant8(x, r, gamma, None, q2, s2, eps=1e-6)
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)
    lb.add_norm_quant8(x, None, gamma, None, q2, s2)
    torch.cuda.synchronize()
    check_norm(q2, s2, true_norm(x.double(), gamma, 0.0))


@pytest.mark.parametrize("xt,rt", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("rows,cols", [(3, 5), (70, 255), (33, 301), (20, 511), (41, 700), (7, 2050), (5, 5001), (3, 17003)])
def test_add_norm_quant8_padding_is_not_read(lb, xt, rt, rows, cols):
    """NaN behind the rows, and rows that start on no boundary, change nothing."""
    x, r = rnd((rows, cols), cols, TYPES[xt]), rnd((rows, cols), cols + 1, TYPES[rt])
    gamma = rnd((1, cols), 7)[0]
    for shift, extra in ((0, -cols % 8), (3, 0)):
        outs = []
        for fill in (in_nan, lambda t, pitch, at: torch.nan_to_num_(in_nan(t, pitch, at)._base, nan=2.0).as_strided(
                t.shape, (pitch, 1), at)):
            xv, rv = fill(x, cols + extra, shift), fill(r, cols + extra, shift)
            q, s, buf = out8(rows, cols)
            lb.add_norm_quant8(xv, rv, gamma, rv, q, s)  # the sum over its residual
            torch.cuda.synchronize()
            assert canary_kept(buf, rows, cols) and torch.isfinite(s).all()
            outs.append((q.view(torch.uint8).clone(), s, rv.clone()))
            assert rv._base[:shift].isnan().all() if fill is in_nan else (rv._base[:shift] == 2.0).all()
        assert all(torch.equal(a, b) for a, b in zip(*outs))
        assert torch.equal(outs[0][2], (x.float() + r.float()).to(TYPES[rt]))


def test_add_norm_quant8_matches_the_trunk_norm(lb):
    """eps = 0 is norm_gates' norm: the 8-bit values are its fp16 values within both roundings."""
    x, gamma = rnd((2294, 256), 1), 1.0 + 0.1 * rnd((1, 256), 2)[0]
    h16 = torch.empty(2294, 256, dtype=torch.float16, device="cuda")
    lb.norm_gates(x, gamma, rnd((8, 256), 3), rnd((1, 8), 4)[0].contiguous(), h16, torch.empty(2294, 8, device="cuda"))
    q, s, _ = out8(2294, 256)
    lb.add_norm_quant8(x, None, gamma, None, q, s)
    lb.op_sync()
    e = expand(s.double(), 2294, 256, 1)
    h = h16.double()
    assert ((q.double() * e - h).abs() <= torch.maximum(h.abs() * 2.0 ** -4, e * 2.0 ** -10) + h.abs() * 2.0 ** -10
            + 2.0 ** -24).all()


@pytest.mark.parametrize("cols", [256, 1000, 2048])
def test_add_norm_quant8_in_place_and_extreme_rows(lb, cols):
    x = rnd((8, cols), 1)
    r = rnd((8, cols), 2)
    x[1], r[1] = 0.0, 0.0                  # nothing to norm
    x[2] *= 1e30                           # the squares overflow 32 bits
    r[2] *= 1e30
    x[3] *= 3e37
    r[3] = 0.0
    x[4] *= 1e-16                          # small, above the norm's floor
    r[4] *= 1e-16
    r[5, 3] = math.inf
    x[6, cols - 1] = math.nan
    x[7] *= 1e-30                          # below the floor: values shrink with it
    r[7] *= 1e-30
    x = x.clamp(-3.0e38, 3.0e38)
    gamma = 1.0 + 0.1 * rnd((1, cols), 3)[0]
    y64 = (x + r).double()  # the fp32 sum
    want = true_norm(y64, gamma, 0.0)
    stream = r.clone()
    q, s, _ = out8(8, cols)
    lb.add_norm_quant8(x, stream, gamma, stream, q, s, eps=0.0)
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(stream, nan=-1.0), torch.nan_to_num(x + r, nan=-1.0))
    keep = [0, 2, 3, 4, 7]
    # the fp32 floor 1e-12 / sqrt(cols) and its quotient are rounded too, inside the bound
    check_norm(q[keep], s[:, keep], want[keep])
    assert (q[1].float() == 0).all() and (s[:, 1] == 2.0 ** -126).all()
    assert torch.isnan(q[5, :128].float()).all() and (q[5, 128:].float() == 0).all()  # infinity: its block only
    assert torch.isnan(q[6].float()).all() and torch.isnan(s[:, 6]).all()
    # x itself as the destination
    x2 = x.clone()
    q2, s2, _ = out8(8, cols)
    lb.add_norm_quant8(x2, r, gamma, x2, q2, s2, eps=0.0)
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8))


# ---- products ------------------------------------------------------------------
def operand(lb, rows, k, br, seed, pad_code=0x7F, scale=1.0):
    """A seeded 8-bit operand whose bytes past column k are NaN codes, and its values in 64 bits."""
    x = rnd((rows, k), seed, scale=scale) * torch.exp(0.5 * rnd((1, k), seed + 1))
    q, s, _ = out8(rows, k, br, code=pad_code)
    lb.quant8(x, q, s, block_rows=br)
    return q, s, q.double() * expand(s.double(), rows, k, br)


def product(a64, w64, k):
    h = a64 @ w64.t()
    tol = (128 + 2 * -(-k // 128) + 8) * 2 * U * (a64.abs() @ w64.abs().t())
    return h, tol


SHAPES = [(1, 1, 1), (1, 16, 16), (1, 128, 128), (1, 129, 250), (1, 1000, 4096), (2, 256, 300), (7, 64, 128),
          (16, 1024, 256), (17, 130, 640), (33, 515, 127), (62, 1024, 256), (62, 256, 1024), (64, 128, 2048), (65, 384, 384),
          (100, 300, 700), (127, 256, 256), (128, 128, 129), (129, 257, 513), (200, 77, 1500), (255, 1536, 256),
          (300, 520, 1000), (558, 1536, 256), (1003, 1000, 777), (2294, 256, 1024), (4097, 130, 130), (2048, 2048, 512),
          # more tiles than SMs: the tiled kernel, from one K-block to many, ragged rows, columns and K
          (9999, 260, 100), (30001, 17, 40), (12000, 33, 900), (9000, 192, 256), (9001, 251, 200), (5000, 700, 129), (2500, 1100, 2100), (19000, 136, 385)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm8(lb, m, n, k):
    a, sa, a64 = operand(lb, m, k, 1, 10 * m + n)
    w, sw, w64 = operand(lb, n, k, 128, 10 * n + k, scale=0.1)
    bias = rnd((1, n), 5)[0]
    h, tol = product(a64, w64, k)
    for i, (kind, with_bias, with_resid, pitch) in enumerate([
            ("f32", True, True, 0), ("f32", False, True, 3), ("f16", True, False, 8), ("f16", False, True, 0),
            ("bf16", True, True, 1), ("bf16", False, False, 0), ("f16", True, True, 2), ("bf16", False, False, 3)]):
        dt = TYPES[kind]
        buf = torch.full((m + 1, n + pitch), 5.0, dtype=dt, device="cuda")
        out = buf[:m, :n]
        # residual rows at the output's pitch, starting one value in where there is room
        resid = rnd((m, n), 6 + i, dt, pad=pitch, shift=min(pitch, i % 2)) if with_resid else None
        lb.gemm8(a, sa, w, sw, out, bias=bias if with_bias else None, resid=resid)
        lb.op_sync()
        want, lim = h, tol
        if with_bias:
            want = want + bias.double()
            lim = lim + -(-k // 128) * U * bias.double().abs()
        if with_resid:
            want = want + resid.double()
        # two fp32 additions, then the rounding to the output's type (fp16: subnormal step 2^-25)
        size = tol + h.abs() + (bias.double().abs() if with_bias else 0) + (resid.double().abs() if with_resid else 0)
        lim = lim + 2 * U * size + (want.abs() + tol) * torch.finfo(dt).eps / 2 + (2.0 ** -25 if kind == "f16" else 0)
        err = (out.double() - want).abs()
        assert (err <= lim).all(), (kind, float((err / lim).max()))
        assert (buf[m] == 5.0).all() and (buf[:, n:] == 5.0).all()


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("with_bias", [True, False])
def test_gemm8_gelu_quant8(lb, m, n, k, with_bias):
    a, sa, a64 = operand(lb, m, k, 1, 10 * m + n)
    w, sw, w64 = operand(lb, n, k, 128, 10 * n + k, scale=1.0 / math.sqrt(k))
    bias = rnd((1, n), 5)[0] if with_bias else None
    h, tol = product(a64, w64, k)
    if with_bias:
        h = h + bias.double()
        tol = tol + U * (h.abs() + tol) + -(-k // 128) * U * bias.double().abs()
    g = 0.5 * h * torch.special.erfc(-h / math.sqrt(2.0))
    tol_g = 1.13 * tol + h.abs() * 2.0 ** -20
    q, s, buf = out8(m, n, pitch=n + 5)
    lb.gemm8_gelu_quant8(a, sa, w, sw, bias, q, s)
    lb.op_sync()
    e = true_scales(g, 1)
    top_tol = true_scales(tol_g, 1)
    assert ((s.double() - e).abs() <= top_tol + e * 2 * U).all()
    check8(q, s, g, 1, tol_g, math.inf)
    assert canary_kept(buf, m, n)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("m,n,k", [(4097, 333, 200), (4130, 262, 70), (300, 333, 200), (33, 70, 300)])
def test_gemm8_rows_at_any_offset(lb, kind, m, n, k):
    """The same bits wherever the rows of the output and the residual start, and nothing beside them is written."""
    dt = TYPES[kind]
    a, sa, _ = out8(m, k)
    w, sw, _ = out8(n, k, 128)
    lb.quant8(rnd((m, k), 1), a, sa)
    lb.quant8(rnd((n, k), 2, scale=k ** -0.5), w, sw, 128)
    bias, r = rnd((1, n), 3)[0].contiguous(), rnd((m, n), 4, dt)
    out = {}
    for with_resid in (False, True):
        out[with_resid] = torch.empty(m, n + -n % 8, dtype=dt, device="cuda")[:, :n]
        lb.gemm8(a, sa, w, sw, out[with_resid], bias=bias, resid=in_nan(r, n + -n % 8, 0) if with_resid else None)
    for shift in range(4):
        for pitch in (n, n + 1, n + 2):
            for rp, rs in ((None, 0), (n, 0), (n, 1), (n + 1, 0), (n + 1, 3)):
                buf = torch.full((m * pitch + shift + 16,), 5.0, dtype=dt, device="cuda")
                view = buf.as_strided((m, n), (pitch, 1), shift)
                lb.gemm8(a, sa, w, sw, view, bias=bias, resid=None if rp is None else in_nan(r, rp, rs))
                torch.cuda.synchronize()
                assert torch.equal(view, out[rp is not None]), (shift, pitch, rp, rs)
                view.fill_(5.0)
                assert (buf == 5.0).all()


@pytest.mark.parametrize("m,n,k", [(5, 200, 300), (300, 520, 1000), (4097, 130, 130), (9000, 200, 300)])
def test_gemm8_adds_into_its_residual(lb, m, n, k):
    a, sa, a64 = operand(lb, m, k, 1, 1)
    w, sw, w64 = operand(lb, n, k, 128, 2)
    x = rnd((m, n), 3)
    h, tol = product(a64, w64, k)
    want = h + x.double()
    got = x.clone()
    lb.gemm8(a, sa, w, sw, got, resid=got)
    lb.op_sync()
    assert ((got.double() - want).abs() <= tol + 2 * U * (h.abs() + x.double().abs() + tol)).all()


@pytest.mark.parametrize("m,n,k", [(9, 300, 520), (400, 300, 520), (6000, 384, 256)])
def test_gemm8_bad_blocks_stay_in_their_rows(lb, m, n, k):
    """A NaN block of A spoils its row, a NaN block of W its 128 columns, nothing else."""
    a, sa, _ = operand(lb, m, k, 1, 1)
    w, sw, _ = operand(lb, n, k, 128, 2)
    clean = torch.empty(m, n, device="cuda")
    lb.gemm8(a, sa, w, sw, clean)
    x = rnd((m, k), 1) * torch.exp(0.5 * rnd((1, k), 2))
    x[3, 130] = math.inf
    lb.quant8(x, a, sa)
    got = torch.empty(m, n, device="cuda")
    lb.gemm8(a, sa, w, sw, got)
    lb.op_sync()
    keep = torch.arange(m, device="cuda") != 3
    assert torch.isnan(got[3]).all() and torch.equal(got[keep], clean[keep])
    sw[1, 1] = math.nan
    lb.gemm8(a, sa, w, sw, got)
    q, s, _ = out8(m, n)
    lb.gemm8_gelu_quant8(a, sa, w, sw, None, q, s)
    lb.op_sync()
    cols = (torch.arange(n, device="cuda") // 128) != 1
    assert torch.isnan(got[:, ~cols]).all() and torch.equal(got[keep][:, cols], clean[keep][:, cols])
    assert torch.isnan(s[1]).all() and torch.isnan(q[:, 128:256].float()).all()
    assert not torch.isnan(s[0][keep]).any() and not torch.isnan(q[keep][:, cols].float()).any()


@pytest.mark.parametrize("m,ld", [(1100, 2 ** 21), (20000, 2 ** 18)])  # split and tiled kernel
def test_gemm8_rows_far_apart(lb, m, ld):
    """Operand, residual and output offsets past 2^31."""
    n, k = 136, 260
    a, sa, a64 = operand(lb, m, k, 1, 1)
    w, sw, w64 = operand(lb, n, k, 128, 2)
    ab = torch.full((m, ld), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, 64:64 + k]
    ab.copy_(a)
    ob = torch.zeros(m, ld, dtype=torch.float16, device="cuda")
    out = ob[:, 8:8 + n]
    h, tol = product(a64, w64, k)
    lb.gemm8(ab, sa, w, sw, out)
    lb.op_sync()
    assert (m - 1) * ld > 2 ** 31
    assert ((out.double() - h).abs() <= tol + (h.abs() + tol) * 2.0 ** -11 + 2.0 ** -25).all()
    assert int(torch.count_nonzero(ob)) == int(torch.count_nonzero(out))
    x = rnd((m, n), 3, torch.float16)
    out.copy_(x)
    lb.gemm8(ab, sa, w, sw, out, resid=out)
    lb.op_sync()
    want = h + x.double()
    lim = tol + 2 * U * (h.abs() + x.double().abs() + tol) + (want.abs() + tol) * 2.0 ** -11 + 2.0 ** -25
    assert ((out.double() - want).abs() <= lim).all()


def test_gemm8_same_bits_every_time(lb):
    for m, n, k in [(1, 1000, 4096), (62, 256, 1024), (300, 520, 1000), (2294, 1536, 256)]:
        a, sa, _ = operand(lb, m, k, 1, 1)
        w, sw, _ = operand(lb, n, k, 128, 2)
        outs = []
        for _ in range(3):
            out = torch.empty(m, n, device="cuda")
            lb.gemm8(a, sa, w, sw, out)
            outs.append(out)
        lb.op_sync()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ---- together --------------------------------------------------------------------
def feed_forward8(lb, b, stream=None):
    """The feed-forward half of a step in 8 bits: norm, FF1 + GELU, FF2 + residual."""
    lb.add_norm_quant8(b["branch"], b["x"], b["gamma"], b["y"], b["h8"], b["h8s"], stream=stream)
    lb.gemm8_gelu_quant8(b["h8"], b["h8s"], b["w1"], b["w1s"], b["b1"], b["g8"], b["g8s"], stream=stream)
    lb.gemm8(b["g8"], b["g8s"], b["w2"], b["w2s"], b["y"], bias=b["b2"], resid=b["y"], stream=stream)


def ff_state(lb, rows, seed):
    b = {"branch": rnd((rows, 256), seed, torch.float16, 0.5), "x": rnd((rows, 256), seed + 1),
         "gamma": 1.0 + 0.1 * rnd((1, 256), seed + 2)[0], "y": torch.empty(rows, 256, device="cuda"),
         "b1": 0.05 * rnd((1, 1024), seed + 3)[0], "b2": 0.02 * rnd((1, 256), seed + 4)[0],
         "w1f": rnd((1024, 256), seed + 5, scale=0.05), "w2f": rnd((256, 1024), seed + 6, scale=0.02)}
    b["h8"], b["h8s"] = lb.empty8(rows, 256)
    b["g8"], b["g8s"] = lb.empty8(rows, 1024)
    b["w1"], b["w1s"] = lb.empty8(1024, 256, 128)
    b["w2"], b["w2s"] = lb.empty8(256, 1024, 128)
    lb.quant8(b["w1f"], b["w1"], b["w1s"], block_rows=128)
    lb.quant8(b["w2f"], b["w2"], b["w2s"], block_rows=128)
    return b


@pytest.mark.parametrize("rows", [1, 62, 558, 16058])
def test_feed_forward_in_8_bits(lb, rows):
    b = ff_state(lb, rows, 40)
    feed_forward8(lb, b)
    lb.op_sync()
    y = (b["branch"].float() + b["x"]).double()
    n = true_norm(y, b["gamma"], 0.0)
    check_norm(b["h8"], b["h8s"], n)
    # the 8-bit values between the launches are what the next launch reads
    w1 = b["w1"].double() * expand(b["w1s"].double(), 1024, 256, 128)
    w2 = b["w2"].double() * expand(b["w2s"].double(), 256, 1024, 128)
    g8 = b["g8"].double() * expand(b["g8s"].double(), rows, 1024, 1)
    h, tol = product(g8, w2, 1024)
    want = h + b["b2"].double() + y
    assert ((b["y"].double() - want).abs() <= tol + 8 * U * b["b2"].double().abs()  # 8 blocks of K = 1024
            + 4 * U * (h.abs() + b["b2"].double().abs() + y.abs() + tol)).all()
    # and the whole beside the fp16 feed-forward of the same weights: each branch value carries relative
    # errors of at most 2^-4 from four quantisations (norm, W1, gelu, W2); their root mean square is below
    # 2^-4 / sqrt(3) each, so the branch is within 4 * 2^-4 of its own size
    h16 = n.to(torch.float16)
    x16 = torch.empty(rows, 256, device="cuda")
    lb.feed_forward(h16, b["w1f"].half(), b["b1"], b["w2f"].half(), b["b2"], y.float(), x16)
    lb.op_sync()
    branch16, branch8 = x16.double() - y, b["y"].double() - y
    assert (branch8 - branch16).norm() <= 0.25 * branch16.norm()


def test_side_stream_and_graph_replays(lb):
    """On a side stream, and captured: two graphs in flight at once give what eager calls give."""
    states = [ff_state(lb, rows, 60 + rows) for rows in (62, 2294)]
    want = []
    for b in states:
        feed_forward8(lb, b)
        want.append(b["y"].clone())
    lb.op_sync()
    streams = [torch.cuda.Stream() for _ in states]
    graphs = []
    for b, st in zip(states, streams):
        b["y"].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            feed_forward8(lb, b, stream=st)
        lb.op_sync(st)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            feed_forward8(lb, b, stream=torch.cuda.current_stream())
        graphs.append(g)
    for b, w in zip(states, want):
        assert torch.equal(b["y"], w)
        b["y"].zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for b, w in zip(states, want):
        assert torch.equal(b["y"], w)
    # a replay reads the inputs of its own time
    states[0]["x"].mul_(-1.0)
    torch.cuda.synchronize()
    graphs[0].replay()
    torch.cuda.synchronize()
    eager = states[0]["y"].clone()
    feed_forward8(lb, states[0])
    lb.op_sync()
    assert torch.equal(eager, states[0]["y"]) and not torch.equal(eager, want[0])


def test_two_products_at_once_on_two_streams(lb):
    """Tiled and split products of different streams in flight together: each as alone, no shared workspace."""
    jobs = []
    for i, (m, n, k) in enumerate([(2294, 1536, 256), (62, 1536, 256), (9000, 520, 300), (1, 4096, 4096)]):
        a, sa, _ = operand(lb, m, k, 1, 10 + i)
        w, sw, _ = operand(lb, n, k, 128, 20 + i)
        want = torch.empty(m, n, device="cuda")
        lb.gemm8(a, sa, w, sw, want)
        jobs.append((a, sa, w, sw, want, torch.zeros_like(want), torch.cuda.Stream()))
    lb.op_sync()
    torch.cuda.synchronize()
    for _ in range(20):
        for a, sa, w, sw, _, out, st in jobs:
            lb.gemm8(a, sa, w, sw, out, stream=st)
    torch.cuda.synchronize()
    for *_, want, out, _ in jobs:
        assert torch.equal(out, want)
    lb.op_sync()


FIRST_CALL_IN_A_CAPTURE = """
import sys
sys.path.insert(0, sys.argv[1])
import torch, lbrr
q, s = lbrr.empty8(4, 128); w, ws = lbrr.empty8(128, 128, 128); out = torch.zeros(4, 128, device="cuda")
x = torch.ones(128, 128, device="cuda")
st = torch.cuda.Stream()
with torch.cuda.stream(st):
    lbrr.quant8(x[:4], q, s, stream=st); lbrr.quant8(x, w, ws, 128, stream=st)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=st):
    try:
        lbrr.gemm8(q, s, w, ws, out, stream=torch.cuda.current_stream())
        raise SystemExit("not refused")
    except lbrr.LbrrError as e:
        assert e.code == lbrr.ERR_STATE and "graph" in str(e), e
    out.add_(1.0)
lbrr.gemm8(q, s, w, ws, out, stream=st)
lbrr.op_sync(st)
assert (out - 128.0).abs().max() < 1e-3, out
g.replay()
torch.cuda.synchronize()
assert (out - 129.0).abs().max() < 1e-3, out
print("ok")
"""


def test_first_product_of_a_process_is_refused_inside_a_capture(tmp_path):
    import subprocess
    import sys
    from pathlib import Path
    pkg = Path(__file__).resolve().parent.parent / "logic-bs-roformer-rs_b200"
    script = tmp_path / "first_call.py"
    script.write_text(FIRST_CALL_IN_A_CAPTURE)
    r = subprocess.run([sys.executable, str(script), str(pkg)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr


# ---- refusals that need device tensors ---------------------------------------------
def test_binding_refusals(lb):
    x = rnd((8, 256), 1)
    q, s, _ = out8(8, 256)
    w, sw, _ = out8(128, 256, 128)
    out = torch.zeros(8, 128, device="cuda")

    def no(fn, word):
        with pytest.raises(lb.LbrrError) as ei:
            fn()
        assert ei.value.code == lb.ERR_INVALID and word in str(ei.value), str(ei.value)

    no(lambda: lb.quant8(x.double(), q, s), "float32")
    no(lambda: lb.quant8(x.t(), q.t(), s), "columns")
    no(lambda: lb.quant8(x, q[:, :255], s), "shape")
    no(lambda: lb.quant8(x, q, s[:1]), "shape")
    no(lambda: lb.quant8(x, q.view(torch.uint8), s), "float8")
    no(lambda: lb.quant8(x, q, s.half()), "float32")
    no(lambda: lb.quant8(x, q[:1].expand(8, 256), s), "overlapping rows")
    no(lambda: lb.quant8(x, q.cpu(), s), "CUDA device")
    g = torch.ones(256, device="cuda")
    no(lambda: lb.add_norm_quant8(x, x.half(), g, None, q, s), "resid")
    no(lambda: lb.add_norm_quant8(x, None, g, x, q, s), "needs resid")
    no(lambda: lb.add_norm_quant8(x, x.clone(), g[:255], None, q, s), "gamma")
    no(lambda: lb.add_norm_quant8(x, x.clone(), g, torch.empty_like(x).half(), q, s), "y must be")
    both = torch.zeros(9, 256, device="cuda")
    no(lambda: lb.add_norm_quant8(both[:8], x, g, both[1:], q, s), "overlaps x")
    no(lambda: lb.add_norm_quant8(x, both[:8], g, both[1:], q, s), "overlaps resid")
    no(lambda: lb.add_norm_quant8(x, None, g, None, q, s, eps=-1.0), "eps")
    no(lambda: lb.gemm8(q, s, w[:, :240], sw, out), "w must have shape")
    no(lambda: lb.gemm8(q, s, w, sw, out[:, :100]), "out must have shape")
    no(lambda: lb.gemm8(q, s, w, sw, out, bias=torch.zeros(127, device="cuda")), "bias")
    no(lambda: lb.gemm8(q, s, w, sw, out, resid=out.half()), "resid")
    no(lambda: lb.gemm8(q, s, w, sw, both[:8, :128], resid=both[1:, :128]), "overlaps")
    narrow = torch.zeros(8, 260, dtype=torch.float8_e4m3fn, device="cuda")
    no(lambda: lb.gemm8(narrow[:, :256], s, w, sw, out), "16-byte")
    no(lambda: lb.gemm8(torch.zeros(8, 272, dtype=torch.float8_e4m3fn, device="cuda")[:, 8:264], s, w, sw, out),
       "16-byte")
    no(lambda: lb.gemm8_gelu_quant8(q, s, w, sw, None, q, s), "q must have shape")
    assert lb.op_sync() is None


def test_empty_calls(lb):
    e = torch.empty(0, 256, device="cuda")
    q, s = lb.empty8(0, 256)
    w, sw, _ = out8(128, 256, 128)
    lb.quant8(e, q, s)
    lb.add_norm_quant8(e, None, torch.ones(256, device="cuda"), None, q, s)
    lb.gemm8(q, s, w, sw, torch.empty(0, 128, device="cuda"))
    lb.gemm8_gelu_quant8(q, s, w, sw, None, *lb.empty8(0, 128))
    lb.op_sync()
