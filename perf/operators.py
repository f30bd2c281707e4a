"""The 8-bit operators of the trunk: what they compute, on which cases, and at what cost.

Four operators carry a transformer step's matrix products in 8-bit floating point (e4m3) with a 32-bit scale for
every block of 128 columns:

  quant8             v -> (q, scales): blocks of 1 x 128 (activations) or 128 x 128 (weights),
                     s = max(|v|) / 448, q = e4m3(v / s); scales are laid out [column block][row block]
  add_norm_quant8    y = x + resid;  n = y / sqrt(mean(y^2) + eps) * gamma;  n -> (q, scales) by 1 x 128
  gemm8              out = A W^T + bias + resid with A [M][K] and W [N][K] in 8 bits, each 128-column block of the
                     product multiplied by its two scales
  gemm8_gelu_quant8  h = A W^T + bias;  gelu(h) -> (q, scales) by 1 x 128

`run` computes them with elementary torch operations in 32 bits (`own` false) or through the library (`own` true).
"""
import math
import os
import sys

import torch

own = False

BLOCK = 128          # columns (and, for weights, rows) that share a scale
E4M3_MAX = 448.0     # largest finite e4m3 value
MIN_SCALE = 2.0 ** -126
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # a feed-forward weight of the checkpoint, laid out once per load
        dict(name="quant8 weight 1024x256", op="quant8", rows=1024, cols=256, block_rows=128, type="f32", pad=0),
        # the gated attention output of a full chunk (1151 frames x 62 bands), before the out-projection
        dict(name="quant8 rows 71362x512", op="quant8", rows=71362, cols=512, block_rows=1, type="f16", pad=0),
        # one frame's 62 band tokens: the smallest call of a streaming caller
        dict(name="norm 62x256", op="add_norm_quant8", rows=62, cols=256, type="f16", resid_type="f32", eps=0.0),
        # the pre-feed-forward norm of a full chunk: half-precision branch, 32-bit residual stream
        dict(name="norm 71362x256", op="add_norm_quant8", rows=71362, cols=256, type="f16", resid_type="f32",
             eps=0.0),
        # a wide stream in bfloat16 whose last block is ragged
        dict(name="norm 4099x5000", op="add_norm_quant8", rows=4099, cols=5000, type="bf16", resid_type="bf16",
             eps=1e-6),
        # one token against a square weight: the weight's bytes are the cost
        dict(name="gemm8 1x4096x4096", op="gemm8", m=1, n=4096, k=4096, type="bf16", bias=False, resid=False),
        # sizes that are multiples of nothing
        dict(name="gemm8 1003x1000x777", op="gemm8", m=1003, n=1000, k=777, type="f32", bias=True, resid=False),
        # the QKV projection of a full chunk
        dict(name="gemm8 71362x1536x256", op="gemm8", m=71362, n=1536, k=256, type="f16", bias=True, resid=False),
        # the second feed-forward projection of a full chunk, onto the residual stream
        dict(name="gemm8 71362x256x1024", op="gemm8", m=71362, n=256, k=1024, type="f32", bias=True, resid=True),
        # a large square product: the tensor cores are the cost
        dict(name="gemm8 8192x8192x8192", op="gemm8", m=8192, n=8192, k=8192, type="bf16", bias=False, resid=False),
        # the first feed-forward projection of one frame and of a full chunk
        dict(name="gelu 62x1024x256", op="gemm8_gelu_quant8", m=62, n=1024, k=256),
        dict(name="gelu 71362x1024x256", op="gemm8_gelu_quant8", m=71362, n=1024, k=256),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quant8", "add_norm_quant8", "gemm8", "gemm8_gelu_quant8"])
    kinds = list(TYPES)
    if op == "quant8":
        cols, kind = _log(rng, 1, 8192), rng.choice(kinds)
        rows = _log(rng, 1, min(71362, 71362 * 512 // (cols * (2 if kind == "f32" else 1))))
        return dict(op=op, rows=rows, cols=cols, block_rows=rng.choice([1, BLOCK]), type=kind,
                    pad=rng.choice([0, 0, 1, 8, 40]))
    if op == "add_norm_quant8":
        cols = _log(rng, 64, 16384)
        rows = _log(rng, 1, min(71362, 60000 * 256 // cols))
        kind = rng.choice(kinds)
        return dict(op=op, rows=rows, cols=cols, type=kind, resid_type=rng.choice([kind, "f32"]),
                    eps=rng.choice([0.0, 1e-6, 1e-5]))
    k, n = _log(rng, 32, 8192), _log(rng, 16, 8192)
    if op == "gemm8":
        m = _log(rng, 1, min(71362, max(1, 71362 * 1536 // max(n, k))))
        return dict(op=op, m=m, n=n, k=k, type=rng.choice(kinds), bias=rng.random() < 0.5, resid=rng.random() < 0.5)
    k, n = min(k, 4096), min(n, 4096)
    m = _log(rng, 1, min(71362, 71362 * 1024 * 256 // (n * k)))
    return dict(op=op, m=m, n=n, k=k)


# ---- inputs -----------------------------------------------------------------
def _blocks(v, block_rows):
    """v [rows][cols], zero-padded to whole blocks: [row blocks][block_rows][column blocks][128]."""
    rows, cols = v.shape
    v = torch.nn.functional.pad(v, (0, -cols % BLOCK, 0, -rows % block_rows))
    return v.view(v.shape[0] // block_rows, block_rows, v.shape[1] // BLOCK, BLOCK)


def _quantise(v, block_rows):
    """v in 32 bits -> (e4m3 [rows][cols], scales [column blocks][row blocks])."""
    rows, cols = v.shape
    b = _blocks(v, block_rows)
    top = b.abs().amax((1, 3))
    s = (top / E4M3_MAX).clamp(min=MIN_SCALE)
    s = torch.where(top < math.inf, s, torch.full_like(s, math.nan))
    q = (b / s[:, None, :, None]).to(E4M3)
    q = q.reshape(q.shape[0] * block_rows, -1)[:rows, :cols]
    return q, s.t().contiguous()


def _held(q):
    """The same values with rows that start on 16-byte boundaries, as the products read them."""
    rows, cols = q.shape
    out = torch.zeros(rows, cols + -cols % 16, dtype=E4M3, device=q.device)[:, :cols]
    out.copy_(q)
    return out


def _space8(rows, cols, block_rows):
    """Space for an 8-bit result and its scales."""
    q = torch.zeros(rows, cols + -cols % 16, dtype=E4M3, device="cuda")[:, :cols]
    return q, torch.zeros(-(-cols // BLOCK), -(-rows // block_rows), device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"op": case["op"]}
    if case["op"] == "quant8":
        rows, cols, kind = case["rows"], case["cols"], TYPES[case["type"]]
        v = randn(rows, cols + case["pad"])
        # weights of the checkpoint's spread; activations with a few loud channels
        v = v * 0.02 if case["block_rows"] == BLOCK else v * torch.exp(0.7 * randn(cols + case["pad"]))
        s["x"] = v.to(kind)[:, :cols]
        s["block_rows"] = case["block_rows"]
        s["q"], s["scales"] = _space8(rows, cols, case["block_rows"])
    elif case["op"] == "add_norm_quant8":
        rows, cols = case["rows"], case["cols"]
        s["x"] = (0.5 * randn(rows, cols)).to(TYPES[case["type"]])
        s["resid"] = (randn(rows, cols) * torch.exp(0.5 * randn(cols))).to(TYPES[case["resid_type"]])
        s["gamma"] = 1.0 + 0.1 * randn(cols)
        s["eps"] = case["eps"]
        s["y"] = torch.zeros(rows, cols, dtype=TYPES[case["resid_type"]], device="cuda")
        s["q"], s["scales"] = _space8(rows, cols, 1)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        a, s["a_scales"] = _quantise(randn(m, k) * torch.exp(0.5 * randn(k)), 1)
        w, s["w_scales"] = _quantise(randn(n, k) / math.sqrt(k), BLOCK)
        s["a"], s["w"] = _held(a), _held(w)
        if case["op"] == "gemm8":
            kind = TYPES[case["type"]]
            s["bias"] = 0.1 * randn(n) if case["bias"] else None
            s["resid"] = randn(m, n).to(kind) if case["resid"] else None
            s["out"] = torch.zeros(m, n, dtype=kind, device="cuda")
        else:
            s["bias"] = 0.1 * randn(n)
            s["q"], s["scales"] = _space8(m, n, 1)
    return s


# ---- one pass ---------------------------------------------------------------
_library = None


def _lbrr():
    global _library
    if _library is None:
        where = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "logic-bs-roformer-rs_b200")
        if where not in sys.path:
            sys.path.insert(0, where)
        import lbrr
        _library = lbrr
    return _library


def _values(q, scales, block_rows):
    """The values an 8-bit tensor stands for, in 32 bits."""
    rows, cols = q.shape
    f = scales.t().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    return q.to(torch.float32) * f


def _gelu(h):
    return 0.5 * h * (1.0 + torch.erf(h * math.sqrt(0.5)))


def run(s):
    op = s["op"]
    if own:
        lbrr, stream = _lbrr(), torch.cuda.current_stream()
        if op == "quant8":
            lbrr.quant8(s["x"], s["q"], s["scales"], block_rows=s["block_rows"], stream=stream)
            return {"q": s["q"], "scales": s["scales"]}
        if op == "add_norm_quant8":
            lbrr.add_norm_quant8(s["x"], s["resid"], s["gamma"], s["y"], s["q"], s["scales"], eps=s["eps"],
                                 stream=stream)
            return {"y": s["y"], "q": s["q"], "scales": s["scales"]}
        if op == "gemm8":
            lbrr.gemm8(s["a"], s["a_scales"], s["w"], s["w_scales"], s["out"], bias=s["bias"], resid=s["resid"],
                       stream=stream)
            return {"out": s["out"]}
        lbrr.gemm8_gelu_quant8(s["a"], s["a_scales"], s["w"], s["w_scales"], s["bias"], s["q"], s["scales"],
                               stream=stream)
        return {"q": s["q"], "scales": s["scales"]}

    if op == "quant8":
        q, scales = _quantise(s["x"].to(torch.float32), s["block_rows"])
        return {"q": q, "scales": scales}
    if op == "add_norm_quant8":
        y = s["x"].to(torch.float32) + s["resid"].to(torch.float32)
        rms = torch.sqrt((y * y).mean(1, keepdim=True) + s["eps"])
        n = y / rms.clamp(min=1e-12 / math.sqrt(y.shape[1])) * s["gamma"]
        q, scales = _quantise(n, 1)
        return {"y": y.to(s["resid"].dtype), "q": q, "scales": scales}
    h = _values(s["a"], s["a_scales"], 1) @ _values(s["w"], s["w_scales"], BLOCK).t()
    if s["bias"] is not None:
        h = h + s["bias"]
    if op == "gemm8":
        if s["resid"] is not None:
            h = h + s["resid"].to(torch.float32)
        return {"out": h.to(s["out"].dtype)}
    q, scales = _quantise(_gelu(h), 1)
    return {"q": q, "scales": scales}


# ---- the definition in 64 bits ----------------------------------------------
def _exact8(v, rows_per_scale):
    """64-bit v -> the unrounded v / s and the scales s, laid out as an 8-bit result is."""
    rows, cols = v.shape
    tops = [part.abs().amax(1) for part in v.split(BLOCK, 1)]
    if rows_per_scale > 1:
        tops = [torch.stack([p.amax() for p in t.split(rows_per_scale)]) for t in tops]
    s = torch.stack(tops).div(E4M3_MAX).clamp(min=MIN_SCALE)
    at_row = torch.arange(rows, device=v.device) // rows_per_scale
    at_col = torch.arange(cols, device=v.device) // BLOCK
    return v / s[at_col][:, at_row].t(), s


def _exact_values(q, scales, rows_per_scale):
    at_row = torch.arange(q.shape[0], device=q.device) // rows_per_scale
    at_col = torch.arange(q.shape[1], device=q.device) // BLOCK
    return q.to(torch.float64) * scales.to(torch.float64)[at_col][:, at_row].t()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant8":
        q, scales = _exact8(s["x"].to(torch.float64), case["block_rows"])
        return {"q": q, "scales": scales}
    if case["op"] == "add_norm_quant8":
        y = s["x"].to(torch.float64) + s["resid"].to(torch.float64)
        length = torch.linalg.vector_norm(y, dim=1, keepdim=True)
        if case["eps"] > 0:
            length = torch.sqrt(length ** 2 + case["eps"] * case["cols"])
        q, scales = _exact8(math.sqrt(case["cols"]) * y / length.clamp(min=1e-12) * s["gamma"].to(torch.float64), 1)
        return {"y": y, "q": q, "scales": scales}
    h = torch.einsum("mk,nk->mn", _exact_values(s["a"], s["a_scales"], 1),
                     _exact_values(s["w"], s["w_scales"], BLOCK))
    if s["bias"] is not None:
        h += s["bias"]
    if case["op"] == "gemm8":
        return {"out": h if s["resid"] is None else h + s["resid"]}
    q, scales = _exact8(0.5 * h * torch.special.erfc(-h / math.sqrt(2.0)), 1)
    return {"q": q, "scales": scales}


# ---- what a pass cannot do without -------------------------------------------
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}

    def held(rows, cols, block_rows):
        return rows * cols + 4 * -(-rows // block_rows) * -(-cols // BLOCK)

    if case["op"] == "quant8":
        n = case["rows"] * case["cols"]
        return {"bytes": n * size[case["type"]] + held(case["rows"], case["cols"], case["block_rows"]),
                "flops": 3 * n}
    if case["op"] == "add_norm_quant8":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size[case["type"]] + 2 * size[case["resid_type"]]) + 4 * case["cols"]
                + held(case["rows"], case["cols"], 1), "flops": 8 * n}
    m, n, k = case["m"], case["n"], case["k"]
    moved = held(m, k, 1) + held(n, k, BLOCK)
    if case["op"] == "gemm8":
        moved += m * n * size[case["type"]] * (2 if case["resid"] else 1) + (4 * n if case["bias"] else 0)
        return {"bytes": moved, "flops": 2 * m * n * k}
    return {"bytes": moved + 4 * n + held(m, n, 1), "flops": 2 * m * n * k + 12 * m * n}
