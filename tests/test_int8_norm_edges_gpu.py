"""The norm where its definition meets the ends of its range: no eps, rows of zeros, rows whose squares
leave fp32."""
import pytest
import torch

from c3_b200 import linear, norm, quant

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
u = 2.0 ** -24

# one size for each kernel: a warp or block per row, on and off the 16-byte grid; the ring (from 32 blocks' worth
# of rows an SM on); two passes
SIZES = [(5, 24), (5, 777), (3, 4096), (10000, 4096), (5000, 1001), (3, 20000)]


@pytest.mark.parametrize("eps", [0.0, 1e-50])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,k", SIZES)
def test_rows_of_zeros_without_eps(cuda_device, m, k, residual, dtype, eps):
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(m + k)
    x = torch.randn((m, k), generator=g, device=dev).to(dtype)
    r = torch.randn((m, k), generator=g, device=dev).to(dtype) if residual else None
    zeros = [0, m // 2, m - 1]
    x[zeros] = 0
    if residual:
        r[zeros] = 0
    w = torch.randn(k, generator=g, device=dev)
    q, scale, h, rstd = norm.rms_norm_int8(x, w, eps, residual=r)
    assert bool((scale[zeros] == 0).all()) and bool((rstd[zeros] == 0).all()) and int(q[zeros].abs().max()) == 0
    rest = torch.ones(m, dtype=torch.bool, device=dev)
    rest[zeros] = False
    hd = h[rest].double()
    want = 1 / torch.sqrt((hd * hd).mean(1))
    adds = 26 + k // 1024  # as in the tests with eps: the root halves the sum's error, four roundings after it
    assert bool(((rstd[rest].double() - want).abs() <= (adds / 2 + 4) * u * want).all())

    # and the gradient of such a row is that of a constant
    dy = torch.randn((m, k), generator=g, device=dev).to(dtype)
    dh = torch.randn((m, k), generator=g, device=dev).to(dtype)
    dx, dw = norm.rms_norm_backward(dy, h, w, rstd, dh=dh)
    assert torch.equal(dx[zeros], dh[zeros])
    xh = h.double() * rstd.double()[:, None]
    ref, size = (dy.double() * xh).sum(0), (dy.double() * xh).abs().sum(0)
    assert bool(((dw.double() - ref).abs() <= (m / 64 + 128) * u * size).all())
    # its row adds nothing to a weight gradient either
    dz = torch.ones((m, 8), dtype=BF16, device=dev)
    assert bool(torch.isfinite(linear.grad_weight_int8(dz, q, scale)).all())


@pytest.mark.parametrize("m,k", [(4, 512), (3, 1001), (2, 20000)])
def test_squares_beyond_fp32(cuda_device, m, k):
    """Documented: the sum of squares is infinite, so rstd and scale are 0; q is still the row's."""
    dev = cuda_device
    x = torch.randn((m, k), generator=torch.Generator(device=dev).manual_seed(k), device=dev)
    w = torch.ones(k, device=dev)
    x[1] *= 1e25
    q, scale, _h, rstd = norm.rms_norm_int8(x, w)
    assert float(rstd[1]) == 0 and float(scale[1]) == 0
    assert torch.equal(q, quant.quantize_rows(x)[0])
    assert float(scale[0]) > 0 and float(rstd[0]) > 0
    x[1] *= 1e-8  # 1e17 and below: in range
    _q, scale, _h, rstd = norm.rms_norm_int8(x, w)
    xd = x.double()
    want = 1 / torch.sqrt((xd * xd).mean(1) + 1e-6)
    assert bool(((rstd.double() - want).abs() <= ((26 + k // 1024) / 2 + 4) * u * want).all())
