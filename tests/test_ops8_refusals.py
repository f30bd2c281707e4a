"""Refusals of the 8-bit operators, without a GPU: every bad argument is named
and refused before any device work, through the C ABI (with addresses that are
never dereferenced) and through the binding's own checks."""
import ctypes as C

import pytest
import torch

import lbrr

P = 0x10000  # a 16-byte aligned address that no call may touch
F32, F16, BF16 = 0, 1, 2


def refused(rc, *words):
    assert rc == lbrr.ERR_INVALID
    msg = lbrr.lib().lbrr_last_error().decode()
    for w in words:
        assert w in msg, msg


QUANT = dict(x=P, x_type=F32, ldx=256, rows=4, cols=256, block_rows=1, q=P, ldq=256, scales=P, lds=4, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "bad x"), (dict(x=P + 2), "bad x"), (dict(ldx=255), "bad x"), (dict(ldx=1 << 40), "bad x"),
    (dict(x_type=3), "x_type"), (dict(x_type=-1), "x_type"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"),
    (dict(cols=0), "cols"), (dict(cols=-5), "cols"), (dict(cols=1 << 24, ldx=1 << 24, ldq=1 << 24), "cols"),
    (dict(block_rows=64), "block_rows"), (dict(block_rows=0), "block_rows"), (dict(q=None), "bad q"),
    (dict(ldq=200), "bad q"), (dict(scales=None), "scales"), (dict(scales=P + 1), "scales"), (dict(lds=3), "scales"),
    (dict(block_rows=128, rows=1 << 30, cols=1 << 20, ldx=1 << 20, ldq=1 << 20, lds=1 << 23), "2^30 blocks")])
def test_quant8(change, word):
    refused(lbrr.lib().lbrr_op_quant8(*{**QUANT, **change}.values()), "lbrr_op_quant8", word)


NORM = dict(x=P, x_type=F16, ldx=256, resid=P, resid_type=F32, ldr=256, gamma=P, eps=0.0, y=P, ldy=256, q=P, ldq=256,
            scales=P, lds=4, rows=4, cols=256, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "bad x"), (dict(x=P + 1), "bad x"), (dict(ldx=100), "bad x"), (dict(x_type=9), "x_type"),
    (dict(resid_type=9), "resid_type"), (dict(resid_type=BF16), "resid_type"),
    (dict(x_type=F32, resid_type=F16), "resid_type"), (dict(ldr=255), "resid"), (dict(resid=P + 2), "resid"),
    (dict(resid=None), "needs resid"), (dict(gamma=None), "gamma"), (dict(gamma=P + 2), "gamma"),
    (dict(eps=-1e-6), "eps"), (dict(eps=2.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(ldy=9), "bad y"),
    (dict(y=P + 2), "bad y"), (dict(q=None), "bad q"), (dict(ldq=255), "bad q"), (dict(lds=3), "scales"),
    (dict(scales=None), "scales"), (dict(rows=-1), "rows"), (dict(cols=0), "32768"), (dict(cols=32769), "32768")])
def test_add_norm_quant8(change, word):
    refused(lbrr.lib().lbrr_op_add_norm_quant8(*{**NORM, **change}.values()), "lbrr_op_add_norm_quant8", word)


@pytest.mark.parametrize("change", [
    dict(), dict(x=2 * P, ldr=512), dict(x_type=F32, resid=2 * P, ldx=512), dict(x_type=F32, resid=2 * P, ldy=512)])
def test_add_norm_quant8_in_place_needs_the_same_rows(change):
    """y at x's or resid's address with another type or another distance between rows."""
    refused(lbrr.lib().lbrr_op_add_norm_quant8(*{**NORM, **change}.values()), "lbrr_op_add_norm_quant8", "in place")


def test_gemm8_in_place_needs_the_same_rows():
    refused(lbrr.lib().lbrr_op_gemm8(*{**GEMM, "ldo": 208}.values()), "lbrr_op_gemm8", "in place")


GEMM = dict(a=P, lda=256, a_scales=P, ldas=8, w=P, ldw=256, w_scales=P, ldws=2, bias=P, resid=P, ldr=200, out=P,
            out_type=F16, ldo=200, m=8, n=200, k=250, stream=None)
GELU = dict(a=P, lda=256, a_scales=P, ldas=8, w=P, ldw=256, w_scales=P, ldws=2, bias=P, q=P, ldq=200, scales=P, lds=8,
            m=8, n=200, k=250, stream=None)
OPERANDS = [
    (dict(a=None), "16-byte"), (dict(a=P + 8), "16-byte"), (dict(lda=250), "16-byte"), (dict(lda=240), "16-byte"),
    (dict(w=None), "16-byte"), (dict(w=P + 1), "16-byte"), (dict(ldw=264), "16-byte"), (dict(a_scales=None), "a_scales"),
    (dict(ldas=7), "a_scales"), (dict(w_scales=None), "w_scales"), (dict(ldws=1), "w_scales"),
    (dict(w_scales=P + 2), "w_scales"), (dict(bias=P + 2), "bias"), (dict(m=-1), "m, n or k"), (dict(n=0), "m, n or k"),
    (dict(k=0), "m, n or k"), (dict(m=(1 << 30) + 1), "m, n or k"), (dict(k=1 << 24), "m, n or k"), (dict(m=1 << 30, n=1 << 15, ldas=1 << 30, ldws=256), "2^30 tiles")]


@pytest.mark.parametrize("change,word", OPERANDS + [
    (dict(out=None), "bad out"), (dict(out=P + 1), "bad out"), (dict(ldo=199), "bad out"), (dict(out_type=4), "out_type"),
    (dict(ldr=199), "bad resid"), (dict(resid=P + 1), "bad resid")])
def test_gemm8(change, word):
    refused(lbrr.lib().lbrr_op_gemm8(*{**GEMM, **change}.values()), "lbrr_op_gemm8", word)


@pytest.mark.parametrize("change,word", OPERANDS + [
    (dict(q=None), "bad q"), (dict(ldq=199), "bad q"), (dict(scales=None), "bad scales"), (dict(lds=7), "bad scales")])
def test_gemm8_gelu_quant8(change, word):
    refused(lbrr.lib().lbrr_op_gemm8_gelu_quant8(*{**GELU, **change}.values()), "lbrr_op_gemm8_gelu_quant8", word)


def test_no_rows_is_no_work():
    L = lbrr.lib()
    assert L.lbrr_op_quant8(*{**QUANT, "rows": 0, "x": None, "q": None}.values()) == lbrr.OK
    assert L.lbrr_op_add_norm_quant8(*{**NORM, "rows": 0, "x": None}.values()) == lbrr.OK
    assert L.lbrr_op_gemm8(*{**GEMM, "m": 0, "a": None, "out": None}.values()) == lbrr.OK
    assert L.lbrr_op_gemm8_gelu_quant8(*{**GELU, "m": 0, "a": None, "q": None}.values()) == lbrr.OK


def binding_refuses(fn, *words):
    with pytest.raises(lbrr.LbrrError) as ei:
        fn()
    assert ei.value.code == lbrr.ERR_INVALID
    for w in words:
        assert w in str(ei.value), str(ei.value)


def test_binding_refuses_host_tensors():
    x = torch.zeros(4, 256)
    q, s = lbrr.empty8(4, 256, device="cpu")
    binding_refuses(lambda: lbrr.quant8(x, q, s), "CUDA device")
    binding_refuses(lambda: lbrr.add_norm_quant8(x, None, torch.ones(256), None, q, s), "CUDA device")
    w, ws = lbrr.empty8(128, 256, 128, device="cpu")
    binding_refuses(lambda: lbrr.gemm8(q, s, w, ws, torch.zeros(4, 128)), "CUDA device")
    binding_refuses(lambda: lbrr.gemm8_gelu_quant8(q, s, w, ws, None, *lbrr.empty8(4, 128, device="cpu")),
                    "CUDA device")


def test_binding_refuses_wrong_ranks_and_blocks():
    q, s = lbrr.empty8(4, 256, device="cpu")
    binding_refuses(lambda: lbrr.quant8(torch.zeros(4), q, s), "matrix")
    binding_refuses(lambda: lbrr.quant8(torch.zeros(4, 256), q, s, block_rows=2), "block_rows")
    binding_refuses(lambda: lbrr.empty8(4, 0, device="cpu"), "cols")
    binding_refuses(lambda: lbrr.empty8(4, 4, 7, device="cpu"), "block_rows")
    binding_refuses(lambda: lbrr.add_norm_quant8(torch.zeros(4), None, None, None, q, s), "matrix")
    binding_refuses(lambda: lbrr.gemm8(q[0], s, q, s, q), "matrices")


def test_empty8_layout():
    q, s = lbrr.empty8(130, 250, 128, device="cpu")
    assert q.shape == (130, 250) and q.stride() == (256, 1) and q.dtype == torch.float8_e4m3fn
    assert s.shape == (2, 2) and s.dtype == torch.float32
    assert lbrr.empty8(130, 250, device="cpu")[1].shape == (2, 130)


def test_signatures_match_the_header():
    """The argument counts the binding declares are the header's."""
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parent.parent / "include" / "lbrr_gpu.h").read_text()
    for name in ("lbrr_op_quant8", "lbrr_op_add_norm_quant8", "lbrr_op_gemm8", "lbrr_op_gemm8_gelu_quant8"):
        args = re.search(r"int %s\(([^)]*)\)" % name, text).group(1).split(",")
        kinds = getattr(lbrr.lib(), name).argtypes
        assert len(args) == len(kinds), name
        for a, k in zip(args, kinds):
            want = C.c_void_p if "*" in a else C.c_int64 if "int64_t" in a else C.c_int32 if "int32_t" in a else C.c_float
            assert k is want, (name, a, k)
