"""Outputs and residuals that are columns of one buffer: what the calls give in buffers of their own, and the columns
beside them unchanged."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lb():
    import lbrr
    lbrr.lib()
    return lbrr


def rnd(shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(62, 256), (3000, 256), (301, 257), (65, 1001), (4, 5000)])
def test_add_norm_quant8(lb, dtype, rows, cols):
    gamma = rnd((cols,), 1)
    buf = rnd((rows, 3 * cols), 2, dtype)
    x, r, y = buf[:, :cols], buf[:, cols:2 * cols], buf[:, 2 * cols:]
    x0, r0, y0 = x.clone(), r.clone(), torch.empty_like(x, memory_format=torch.contiguous_format)
    q0, s0 = lb.empty8(rows, cols)
    q, s = lb.empty8(rows, cols)
    lb.add_norm_quant8(x0, r0, gamma, y0, q0, s0, eps=1e-6)
    lb.add_norm_quant8(x, r, gamma, y, q, s, eps=1e-6)
    torch.cuda.synchronize()
    assert torch.equal(y, y0) and torch.equal(x, x0) and torch.equal(r, r0)
    # rows on other boundaries take another path, whose sums may round otherwise
    if (cols * buf.element_size()) % 16 == 0:
        assert torch.equal(q.view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s, s0)
    else:
        assert ((s - s0).abs() <= s0 * 2.0 ** -20).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(62, 256, 300), (6000, 256, 128), (4097, 131, 200), (33, 77, 100)])
def test_gemm8(lb, dtype, m, n, k):
    a, sa = lb.empty8(m, k)
    w, sw = lb.empty8(n, k, 128)
    lb.quant8(rnd((m, k), 1), a, sa)
    lb.quant8(rnd((n, k), 2), w, sw, block_rows=128)
    buf = rnd((m, 2 * n), 3, dtype)
    for out, resid in ((buf[:, :n], buf[:, n:]), (buf[:, n:], buf[:, :n])):
        r0, want = resid.clone(), torch.empty(m, n, dtype=dtype, device="cuda")
        lb.gemm8(a, sa, w, sw, want, resid=r0)
        lb.gemm8(a, sa, w, sw, out, resid=resid)
        lb.op_sync()
        assert torch.equal(out, want) and torch.equal(resid, r0)
