"""The norm's gradient on rows of 8193 elements and more, where its kernel changes: rows on the
16-byte grid that still fit a ring of buffers, and longer ones; one block, fewer blocks than SMs, and
several rows a block. References, bounds and their reasons are those of test_int8_rows_gpu.py (a
thread now adds 16 pairs of columns in sequence, within the same count)."""
import pytest
import torch

from c3_b200 import norm
from tests.test_int8_rows_gpu import BF16, F32, _bwd_inputs, _check_bwd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dh", [False, True])
@pytest.mark.parametrize("m,k", [(1, 8200), (4, 12288), (5, 8208), (148, 9384), (149, 16384), (600, 12288), (600, 8200),
                                 (300, 14080), (40, 16392), (20, 18000)])
def test_wide_rows(cuda_device, m, k, dh, dtype):
    a = _bwd_inputs(m, k, dtype, dh, cuda_device, m + k)
    dx, dw = norm.rms_norm_backward(*a[:4], dh=a[4])
    _check_bwd(*a, dx, dw)
    dx2, dw2 = norm.rms_norm_backward(*a[:4], dh=a[4])
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


@pytest.mark.parametrize("dtype,k", [(BF16, 12288), (BF16, 16384), (F32, 8704)])
def test_wide_rows_strided_in_place_and_neighbours(cuda_device, dtype, k):
    dev = cuda_device
    m = 310
    dy, h, w, rstd, d = _bwd_inputs(m, k, dtype, True, dev, k)
    want = norm.rms_norm_backward(dy, h, w, rstd, dh=d)
    wide = [torch.full((m + 2, k + 16), 7.0, dtype=dtype, device=dev) for _ in range(3)]
    views = [b[1:1 + m, 8:8 + k] for b in wide]
    for v, t in zip(views, (dy, h, d)):
        v.copy_(t)
    for out in (2, 1, 0):  # each destroys one that the next does not write
        t = [v.clone() for v in views]
        dx, dw = norm.rms_norm_backward(t[0], t[1], w, rstd, dh=t[2], dx=t[out])
        assert dx is t[out] and torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    dx, dw = norm.rms_norm_backward(views[0], views[1], w, rstd, dh=views[2], dx=views[2])
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    views[2].fill_(7.0)
    assert bool((wide[2] == 7).all())


def test_wide_row_that_is_not_finite(cuda_device):
    dy, h, w, rstd, d = _bwd_inputs(300, 12288, BF16, True, cuda_device, 1)
    h[7, 100] = float("inf")
    rstd[7] = 0
    dx, dw = norm.rms_norm_backward(dy, h, w, rstd, dh=d)
    assert bool(torch.isnan(dx[7, 100])) and bool(torch.isfinite(dx[[6, 8]]).all()) and bool(torch.isnan(dw[100]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dh", [False, True])
@pytest.mark.parametrize("m,k", [(148, 8193), (300, 9001), (400, 12287), (149, 16383), (150, 16385)])
def test_wide_rows_off_the_16_byte_grid(cuda_device, m, k, dh, dtype):
    dev = cuda_device
    dy, h, w, rstd, d = _bwd_inputs(m, k, dtype, dh, dev, m + k)
    want = norm.rms_norm_backward(dy, h, w, rstd, dh=d)
    _check_bwd(dy, h, w, rstd, d, *want)
    # rows that start anywhere, with other values around them, and dx over one of the inputs
    wide = [torch.full((m, k + 13), 7.0, dtype=dtype, device=dev) for _ in range(3)]
    views = [b[:, c:c + k] for b, c in zip(wide, (5, 1, 9))]
    for v, t in zip(views, (dy, h, d)):
        if t is not None:
            v.copy_(t)
    dx, dw = norm.rms_norm_backward(views[0], views[1], w, rstd, dh=views[2] if dh else None, dx=views[0])
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    assert torch.equal(views[1], h) and (not dh or torch.equal(views[2], d))
    views[0].fill_(7.0)
    assert bool((wide[0] == 7).all())
