"""What a refused or failed call of the 8-bit operators leaves behind: nothing.  The next call does not report an earlier
one's error, and captures under way elsewhere stay whole.  Each case needs a process of its own, whose first product has
not been called yet."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PKG = Path(__file__).resolve().parent.parent / "logic-bs-roformer-rs_b200"

SETUP = """
import ctypes as C, sys
sys.path.insert(0, sys.argv[1])
import torch, lbrr
rt = C.CDLL("libcudart.so.12")
q, s = lbrr.empty8(4, 128); w, ws = lbrr.empty8(128, 128, 128); out = torch.zeros(4, 128, device="cuda")
x = torch.ones(128, 128, device="cuda")
st = torch.cuda.Stream()
def quantise():
    lbrr.quant8(x[:4], q, s, stream=st); lbrr.quant8(x, w, ws, 128, stream=st)
def product(stream=st):
    lbrr.gemm8(q, s, w, ws, out, stream=stream)
def right():
    torch.cuda.synchronize(); lbrr.op_sync(st)
    assert (out - 128.0).abs().max() < 1e-3, out
def refused(code, fn):
    try:
        fn()
    except lbrr.LbrrError as e:
        assert e.code == code, e
        return str(e)
    raise SystemExit("not refused")
class Blocking:
    '''A capture on a stream that the legacy default stream waits for.'''
    def __enter__(self):
        self.st = C.c_void_p()
        assert rt.cudaStreamCreate(C.byref(self.st)) == 0
        assert rt.cudaStreamBeginCapture(self.st, 2) == 0
    def __exit__(self, *exc):
        g = C.c_void_p()
        self.rc = rt.cudaStreamEndCapture(self.st, C.byref(g))
        if self.rc == 0 and g:
            assert rt.cudaGraphDestroy(g) == 0
        else:
            rt.cudaGetLastError()  # this call's own
        assert rt.cudaStreamDestroy(self.st) == 0
torch.cuda.synchronize()
"""

CASES = {
    # the default stream cannot be asked whether it is capturing while a blocking stream is
    "refused_beside_a_blocking_capture": """
quantise(); torch.cuda.synchronize()
c = Blocking()
with c:
    refused(lbrr.ERR_STATE, lambda: product(None))
assert c.rc == 0
quantise()
product(); right()
""",
    # the first product of the process while another stream is being captured: that capture is not its business
    "first_product_beside_a_capture": """
quantise(); torch.cuda.synchronize()
other, y = torch.cuda.Stream(), torch.zeros(8, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=other):
    y.add_(1.0)
    product()
    y.add_(1.0)
right()
g.replay(); torch.cuda.synchronize()
assert (y == 2.0).all()
""",
    # a launch that fails on the host is reported once
    "failed_launch": """
quantise(); product(); right()
c = Blocking()
with c:
    refused(lbrr.ERR_CUDA, lambda: product(None))
out.zero_(); torch.cuda.synchronize()
quantise()
product(); right()
""",
}


@pytest.mark.parametrize("case", list(CASES))
def test_leaves_nothing_behind(tmp_path, case):
    script = tmp_path / "case.py"
    script.write_text(SETUP + CASES[case] + '\nprint("ok")\n')
    r = subprocess.run([sys.executable, str(script), str(PKG)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr
