"""How exact the weight gradient from an 8-bit checkpoint is: q takes part exactly, dZ * scale to 2^-11 at
least (fp16 in large tiles, two bf16 terms in small ones), sums are fp32 and the output is rounded once.
In large tiles each column of dZ * scale is brought into fp16's range by a power of two of its own, so its
size does not matter, nor that of its neighbours."""
import contextlib

import pytest
import torch

from c3_b200 import _lib, linear, quant

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
u = 2.0 ** -24


@contextlib.contextmanager
def _large_tiles(on):
    """With a cap on its CTAs the call takes the persistent kernel of large tiles, whatever the size."""
    lib = _lib.load()
    lib.c3cu_set_gemm_max_ctas(148 if on else 0)
    try:
        yield
    finally:
        lib.c3cu_set_gemm_max_ctas(0)


@contextlib.contextmanager
def _form(tile, split, ready):
    lib = _lib.load()
    _lib.check(lib.c3cu_set_int8_form(tile, split, ready), "c3cu_set_int8_form")
    try:
        yield
    finally:
        lib.c3cu_set_int8_form(-1, 1, 0)


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _case(m, n, k, dev, seed):
    x = torch.randn((m, k), generator=_gen(dev, seed), device=dev)
    x *= torch.exp(torch.randn(m, 1, generator=_gen(dev, seed + 1), device=dev))
    dz = torch.zeros((m, (n + 7) // 8 * 8), dtype=BF16, device=dev)[:, :n]
    dz.copy_(torch.randn((m, n), generator=_gen(dev, seed + 2), device=dev) * 1e-3)
    q, s = quant.quantize_rows(x)
    return dz, q, s


def _ref(dz, q, s):
    """dW in fp64, the sum of the products' magnitudes, and 2^-39 of each column's largest |dZ * scale|
    times the sum of |q|: what fp16 loses of elements 2^-28 below that largest."""
    z = dz.double() * s.double()[:, None]
    qd = q.double()
    ref = z.t() @ qd
    size = z.abs().t() @ qd.abs()
    far = 2.0 ** -39 * z.abs().amax(0)[:, None] * qd.abs().sum(0)[None, :]
    return ref, size, far


def _check(dw, dz, q, s):
    ref, size, far = _ref(dz, q, s)
    m = dz.shape[0]
    # the output's rounding; the operand's, with fl32(dZ * scale) before it; fp32 sums whose adds may
    # truncate (2 u each, two terms for each product in small tiles)
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -11 + u + (4 * m + 2) * u) * size + far
    assert bool(((dw.double() - ref).abs() <= tol).all())
    return ref


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("m", [1, 2, 5, 64, 130])
@pytest.mark.parametrize("n,k", [(8, 16), (40, 300), (100, 130), (264, 784)])
def test_few_rows(cuda_device, m, n, k, large):
    """With few rows nothing averages out: two roundings to bf16 would show in single elements."""
    dz, q, s = _case(m, n, k, cuda_device, m + n + k)
    with _large_tiles(large):
        dw = linear.grad_weight_int8(dz, q, s)
    _check(dw, dz, q, s)


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("m,n,k", [(128, 256, 784), (997, 56, 233), (776, 56, 2464), (2048, 1024, 1024), (4096, 512, 512),
                                   (640, 2560, 2048)])
def test_the_error_is_the_output_rounding(cuda_device, m, n, k, large):
    """An operand's rounding of 2^-11 is a quarter of the output's at most, both uniform, and
    independent: sqrt(1 + 1/16) = 1.03 of the output's error together."""
    dz, q, s = _case(m, n, k, cuda_device, 3)
    with _large_tiles(large):
        dw = linear.grad_weight_int8(dz, q, s)
        again = linear.grad_weight_int8(dz, q, s)
    ref = _check(dw, dz, q, s)
    least = (ref.to(torch.float32).to(BF16).double() - ref).norm()
    assert float((dw.double() - ref).norm()) <= 1.05 * float(least)
    assert torch.equal(dw, again)


@pytest.mark.parametrize("ready", [0, 1])
@pytest.mark.parametrize("tile", [32, 64, 128])
@pytest.mark.parametrize("split", [1, 2, 4, 8])
def test_every_small_form(cuda_device, tile, split, ready):
    """Sizes off every tile's, and sums of fewer blocks than the cluster has CTAs."""
    dev = cuda_device
    for m, n, k in ((1, 8, 1), (63, 130, 127), (129, 96, 257), (500, 264, 130), (1100, 40, 300)):
        dz, q, s = _case(m, n, k, dev, m + n)
        buf = torch.full((n + 1, k + 5), 7.0, dtype=BF16, device=dev)
        with _form(tile, split, ready):
            dw = linear.grad_weight_int8(dz, q, s, dW=buf[:n, 3:3 + k])
            again = linear.grad_weight_int8(dz, q, s)
        _check(dw, dz, q, s)
        assert torch.equal(dw, again)
        assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 3 + k:] == 7).all()) and bool((buf[n] == 7).all())


def test_training_batch(cuda_device):
    """The large form without a cap."""
    dz, q, s = _case(8192, 4096, 4096, cuda_device, 5)
    dw = linear.grad_weight_int8(dz, q, s)
    ref = _check(dw, dz, q, s)
    least = (ref.to(torch.float32).to(BF16).double() - ref).norm()
    assert float((dw.double() - ref).norm()) <= 1.05 * float(least)


FORMS = [(0, 1, 0), (32, 1, 0), (64, 2, 0), (128, 4, 0), (32, 2, 1), (64, 1, 1), (128, 2, 1)]


@pytest.mark.parametrize("m", [300, 1300])
@pytest.mark.parametrize("form", FORMS)
def test_columns_and_rows_of_any_size(cuda_device, form, m):
    """Columns of dZ from 1e-30 to 1e30 beside each other, one of zeros, rows of X from 1e-6 to 1e6: each
    row of dW is as exact as if it were alone."""
    dev = cuda_device
    n, k = 72, 200
    dz, q, s = _case(m, n, k, dev, 9)
    sizes = 10.0 ** torch.linspace(-30, 30, n, dtype=torch.float64, device=dev)
    dz.copy_((dz.double() * 1e3 * sizes[None, :]).to(BF16))
    dz[:, 5] = 0
    s *= (10.0 ** torch.linspace(-6, 6, m, dtype=torch.float64, device=dev)).float()
    with _form(*form):
        dw = linear.grad_weight_int8(dz, q, s)
    _check(dw, dz, q, s)
    assert bool((dw[5] == 0).all())


@pytest.mark.parametrize("form", FORMS)
def test_products_at_the_ends_of_fp32(cuda_device, form):
    """Products below fp32's normal numbers are held to half of a fixed unit. Large tiles: fl32(dZ * scale)
    is a multiple of 2^-149. Small tiles: three bf16 of the product times 2^6 (head, what it
    leaves, tail), whose last place below 2^-126 is 2^-133, are rounded to half of that at most, so the
    product is held to 3 * 2^-134 / 2^6 < 2^-138."""
    dev = cuda_device
    m, n, k = 70, 16, 40
    dz, q, s = _case(m, n, k, dev, 11)
    tiny = (dz.double() * 2.0 ** -120).to(BF16)
    with _form(*form):
        dw = linear.grad_weight_int8(tiny, q, s)
    ref, size, far = _ref(tiny, q, s)
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -11 + (4 * m + 3) * u) * size + far + 2.0 ** -133
    tol = tol + (2.0 ** -149 if form[0] == 0 or form[2] else 2.0 ** -138) * q.double().abs().sum(0)
    assert bool(((dw.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("m", [130, 1300])
@pytest.mark.parametrize("form", FORMS)
def test_what_is_not_finite_stays_so_and_where_it_is(cuda_device, form, m):
    dev = cuda_device
    n, k = 40, 96
    dz, q, s = _case(m, n, k, dev, 13)
    clean = dz.clone()
    q[q == 0] = 1
    dz[7, 3] = float("inf")  # the rows of a few blocks apart: one alone meets it
    dz[9, 4] = float("nan")
    with _form(*form):
        dw = linear.grad_weight_int8(dz, q, s)
    assert torch.equal(dw[3], (q[7].float() * float("inf")).to(BF16))  # infinity times a number that is not zero
    assert bool(torch.isnan(dw[4]).all())
    dz[7, 3] = dz[9, 4] = clean[7, 3] * 0
    rest = [i for i in range(n) if i not in (3, 4)]
    _check(dw[rest], dz[:, rest], q, s)


@pytest.mark.parametrize("form", FORMS)
def test_large_products(cuda_device, form):
    """Products of dZ and scale up to 2^121 (small tiles take them times 2^6), in sums that fp32 holds."""
    dev = cuda_device
    m, n, k = 66, 16, 24
    dz = torch.zeros((m, n), dtype=BF16, device=dev)
    dz[3], dz[65] = 1.5 * 2.0 ** 100, -2.0 ** 100
    q = quant.empty_rows(m, k, dev)
    q.fill_(127)
    q[3] = (torch.arange(k, device=dev) % 7 - 3).to(torch.int8)
    q[65] = 2
    s = torch.full((m,), 2.0 ** 20, device=dev)
    with _form(*form):
        dw = linear.grad_weight_int8(dz, q, s)
    want = (1.5 * q[3].double() - 2) * 2.0 ** 120  # exact in bf16
    assert torch.equal(dw.double(), want.expand(n, k))
