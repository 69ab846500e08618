"""The 8-bit path on matrices of more than 2^31 elements: what the last rows give is what they give
alone. 600000 x 4096 (2.46e9 elements)."""
import pytest
import torch

from c3_b200 import linear, norm, quant
from tests.test_int8_rows_gpu import BF16, F32, _bwd_ref, u

pytestmark = pytest.mark.gpu

M, K, LAST = 600_000, 4096, 40


@pytest.fixture(scope="module")
def x(cuda_device):
    free, _total = torch.cuda.mem_get_info()
    if free < 40 * 2 ** 30:
        pytest.skip("needs 40 GB")
    t = torch.zeros((M, K), dtype=BF16, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    t[-LAST:] = torch.randn((LAST, K), generator=g, device=cuda_device).to(BF16)
    t[0] = 1.0
    return t


def test_rows(x):
    dev = x.device
    q, s = quant.quantize_rows(x)
    q1, s1 = quant.quantize_rows(x[-LAST:].clone())
    assert torch.equal(q[-LAST:], q1) and torch.equal(s[-LAST:], s1)
    assert bool((q[1:-LAST] == 0).all()) and bool((s[1:-LAST] == 0).all()) and bool((q[0] == 127).all())
    del q
    w = torch.ones(K, device=dev)
    q, s, h, rstd = norm.rms_norm_int8(x, w, residual=x)
    assert torch.equal(h[-LAST:], 2 * x[-LAST:])
    q1, s1, _h1, rstd1 = norm.rms_norm_int8(x[-LAST:].clone(), w, residual=x[-LAST:].clone())
    # q does not depend on rstd; rstd's sums may be taken in another order (36 additions, u each, halved by the root)
    assert torch.equal(q[-LAST:], q1) and bool(((rstd[-LAST:] - rstd1).abs() <= 40 * u * rstd1).all())
    del q, s, h
    dx, dw = norm.rms_norm_backward(x, x, w, rstd)
    rx, size, rw, rsize = _bwd_ref(x[-LAST:], x[-LAST:], w, rstd[-LAST:], None)
    tol = 2.0 ** -8 * rx.abs() + 40 * u * size
    assert bool(((dx[-LAST:].double() - rx).abs() <= tol).all())
    rw0 = (x[0].double() ** 2) * rstd[0].double()  # the one other row that is not zero
    # all but these rows add zeros: at most LAST + 1 additions round, and the products before them
    assert bool(((dw.double() - rw - rw0).abs() <= (LAST + 8) * u * (rsize + rw0)).all())


@pytest.mark.parametrize("n", [64, 4096])
def test_linear_tokens(x, n):
    dev = x.device
    g = torch.Generator(device=dev).manual_seed(2)
    q, s = quant.quantize_rows(x)
    wq, ws = quant.quantize_rows(torch.randn((n, K), generator=g, device=dev))
    b = torch.randn(n, generator=g, device=dev)
    y, mask = linear.forward_int8(q, s, wq, ws, b)
    y1, mask1 = linear.forward_int8(q[-LAST:].clone(), s[-LAST:].clone(), wq, ws, b)
    assert torch.equal(y[-LAST:], y1) and torch.equal(mask[-LAST:], mask1)
    assert torch.equal(y[1], b.clamp_min(0).to(BF16))


@pytest.mark.parametrize("m", [1, 2, 8])
def test_linear_channels(x, m):
    """The large matrix as the weights."""
    wq, ws = quant.quantize_rows(x)
    xq, xs = quant.quantize_rows(x[-m:].clone())
    y, mask = linear.forward_int8(xq, xs, wq, ws, out_dtype=F32)
    y1, _ = linear.forward_int8(xq, xs, wq[-64:].clone(), ws[-64:].clone(), out_dtype=F32)
    assert torch.equal(y[:, -64:], y1) and bool((y[:, 1:-64] == 0).all()) and bool((mask[:, 1:-2] == 0).all())


@pytest.mark.parametrize("n", [16, 512])
def test_weight_gradient(x, n):
    dev = x.device
    g = torch.Generator(device=dev).manual_seed(3)
    q, _s = quant.quantize_rows(x)
    s = torch.ones(M, device=dev)
    dz = torch.zeros((M, n), dtype=BF16, device=dev)
    dz[-LAST:] = torch.randint(-2, 3, (LAST, n), generator=g, device=dev).to(BF16)
    dw = linear.grad_weight_int8(dz, q, s)
    want = (dz[-LAST:].double().t() @ q[-LAST:].double()).to(F32).to(BF16)
    assert torch.equal(dw, want)
