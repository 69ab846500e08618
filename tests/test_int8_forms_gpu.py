"""Every form of the two int8 GEMMs, chosen by hand (c3cu_set_int8_form): each kernel, tile and split, each type
of output, with and without ReLU, mask and bias, at sizes off the tiles', with clusters whose last CTAs have
no part of the sum. The forward's bits and the exact sums of dW do not depend on the form."""
import contextlib

import pytest
import torch

import c3_b200
from c3_b200 import _lib, linear
from tests.test_int8_linear_gpu import BF16, F32, _dw_exact, _forward_ref, _gen, _rows, _unpack

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def _form(tile, split=1, ready=0):
    lib = _lib.load()
    _lib.check(lib.c3cu_set_int8_form(tile, split, ready), "c3cu_set_int8_form")
    try:
        yield
    finally:
        lib.c3cu_set_int8_form(-1, 1, 0)


FORWARD = [(0, 1)] + [(t, s) for t in (16, 32, 64, 128, 256) for s in (1, 2, 4, 8)]
SIZES = [(1, 5, 1), (17, 130, 127), (129, 257, 700), (257, 515, 1032), (300, 33, 129), (520, 300, 48)]


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("tile,split", FORWARD)
def test_forward(cuda_device, tile, split, out_dtype):
    dev = cuda_device
    for m, n, k in SIZES:
        xq, xs = _rows(m, k, dev, m)
        wq, ws = _rows(n, k, dev, n)
        b = torch.randn(n, generator=_gen(dev, 3), device=dev)
        for relu in (True, False):
            for bias in (b, None):
                ref, bits = _forward_ref(xq, xs, wq, ws, bias, relu)
                with _form(tile, split):
                    y, mask = linear.forward_int8(xq, xs, wq, ws, bias, relu=relu, out_dtype=out_dtype)
                assert torch.equal(y, ref.to(out_dtype)), (m, n, k, relu)
                if relu:
                    got, beyond = _unpack(mask, n)
                    assert torch.equal(got, bits) and not bool(beyond.any())
                    with _form(tile, split):
                        y2, none = linear.forward_int8(xq, xs, wq, ws, bias, out_dtype=out_dtype, save_mask=False)
                    assert none is None and torch.equal(y2, y)


@pytest.mark.parametrize("tile,split", FORWARD)
def test_forward_between_neighbours_and_not_finite(cuda_device, tile, split):
    dev = cuda_device
    m, n, k = 261, 200, 208
    xw, xs = _rows(m, 512, dev, 1)
    ww, ws = _rows(n, 512, dev, 2)
    xq, wq = xw[:, 16:16 + k], ww[:, 64:64 + k]
    xs[7], ws[9] = float("nan"), float("inf")
    want, wbits = _forward_ref(xq, xs, wq, ws, None, False)
    ybuf = torch.full((m, n + 24), 5.0, dtype=BF16, device=dev)
    mbuf = torch.full((m, 9), -7, dtype=torch.int32, device=dev)
    with _form(tile, split):
        y, mask = linear.forward_int8(xq, xs, wq, ws, Y=ybuf[:, 8:8 + n], mask=mbuf[:, 1:8])
    assert bool(torch.isnan(y[7]).all())
    same = torch.where(torch.isnan(want), want, want.clamp_min(0)).to(BF16)
    assert torch.equal(torch.nan_to_num(y, nan=-1.0), torch.nan_to_num(same, nan=-1.0))
    assert torch.equal(_unpack(mask, n)[0], wbits)
    assert bool((ybuf[:, :8] == 5).all()) and bool((ybuf[:, 8 + n:] == 5).all())
    assert bool((mbuf[:, 0] == -7).all()) and bool((mbuf[:, 8] == -7).all())


@pytest.mark.parametrize("tile,split", FORWARD)
def test_forward_largest_sums(cuda_device, tile, split):
    dev = cuda_device
    k = linear.INT8_MAX_K
    xq, wq = torch.full((3, 131072), -128, dtype=torch.int8, device=dev)[:, :k], torch.full((2, 131072), -128,
                                                                                            dtype=torch.int8, device=dev)[:, :k]
    one = torch.ones(3, device=dev)
    with _form(tile, split):
        y, _ = linear.forward_int8(xq, one, wq, one[:2].clone(), relu=False, out_dtype=F32)
    assert bool((y == float(torch.tensor(2 ** 14 * k, dtype=torch.float64).float())).all())


DW = [(0, 1, 0)] + [(t, s, r) for t in (32, 64, 128) for s in (1, 2, 4, 8) for r in (0, 1)]


@pytest.mark.parametrize("tile,split,ready", DW)
def test_dw(cuda_device, tile, split, ready):
    dev = cuda_device
    for m, n, k in ((1, 8, 1), (65, 16, 130), (130, 264, 257), (700, 88, 520), (1500, 600, 300)):
        dz, q, s, want = _dw_exact(m, n, k, dev, m + n)
        with _form(tile, split, ready):
            assert torch.equal(linear.grad_weight_int8(dz, q, s), want), (m, n, k)
        q[m // 2], s[m // 2] = 0, float("nan")
        with _form(tile, split, ready):
            assert bool(torch.isnan(linear.grad_weight_int8(dz, q, s)).all())


def test_forms_that_are_not_there(cuda_device):
    dev = cuda_device
    lib = _lib.load()
    for tile, split in ((8, 1), (48, 1), (512, 1), (64, 3), (64, 16), (64, 0), (-2, 1)):
        assert lib.c3cu_set_int8_form(tile, split, 0) == -1
    dz, q, s, want = _dw_exact(70, 16, 40, dev, 1)
    for tile in (16, 256):
        with _form(tile), pytest.raises(c3_b200.C3CUError) as e:
            linear.grad_weight_int8(dz, q, s)
        assert e.value.code == -1
    assert torch.equal(linear.grad_weight_int8(dz, q, s), want)
