"""The row-wise kernels of the 8-bit activation path (quantised rows, RMS norm to int8, its
gradient) against plain fp64 computations.

q is compared for equality: it is defined as the rounding of a real quotient. u = 2^-24 is half
the spacing of fp32 at 1. The fp32 sums have at most 16 sequential and 10 tree additions per row
in the one-pass kernels (K / 1024 sequential ones for long rows), hence the factors below."""
import pytest
import torch

from c3_b200 import norm, quant

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
u = 2.0 ** -24
EPS = 1e-6


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _x(m, k, dtype, seed, dev):
    g = _gen(dev, seed)
    x = torch.randn((m, k), generator=g, device=dev) * torch.exp(torch.randn(k, generator=g, device=dev))
    return x.to(dtype)


def _q_ref(a):
    """Nearest integer to 127 a / A in fp64; a exact in fp64. A row of zeros gives zeros."""
    a = a.double()
    big = a.abs().amax(1, keepdim=True)
    return torch.where(big > 0, torch.round(127 * a / big), 0.0).to(torch.int8), big[:, 0]


def _by_127(big):
    """fl32(A / 127): the fp64 quotient rounded again is the same (53 >= 2 * 24 + 2 bits). torch
    divides fp32 tensors by a number through its reciprocal, which rounds twice."""
    return (big.double() / 127).float()


SIZES = [(1, 1), (1, 2), (3, 7), (5, 16), (2, 31), (9, 128), (4, 255), (130, 512), (7, 513), (33, 777), (3, 1000),
         (17, 4096), (1, 4096), (2, 4104), (1, 8192), (3, 12001), (2, 16384), (2, 16400), (2, 20001), (1, 70000)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k", SIZES)
def test_quantize_rows_is_the_nearest_integer(cuda_device, m, k, dtype):
    x = _x(m, k, dtype, 31 * m + k, cuda_device)
    q, scale = quant.quantize_rows(x)
    ref, big = _q_ref(x)
    assert q.shape == (m, k) and torch.equal(q, ref)
    assert torch.equal(scale, _by_127(big))
    assert q.stride(0) % 16 == 0 or m == 1


def test_quantize_rows_ties_and_extremes(cuda_device):
    """Exact ties go to the even integer; magnitudes at both ends of fp32; zeros of both signs."""
    dev = cuda_device
    ties = torch.arange(-254, 255, device=dev).float()  # 127 x / 254 = x / 2
    rows = [ties * s for s in (1.0, 2.0 ** 100, 2.0 ** -100, 2.0 ** -125, 2.0 ** -140)]
    rows += [torch.full_like(ties, -0.0), torch.full_like(ties, 3e38), torch.full_like(ties, 1e-45)]
    x = torch.stack(rows)
    q, scale = quant.quantize_rows(x)
    ref, big = _q_ref(x)
    assert torch.equal(q, ref)
    assert torch.equal(scale, _by_127(big))
    assert int(q[0, 254 + 1]) == 0 and int(q[0, 254 + 3]) == 2 and int(q[0, 0]) == -127
    # adjacent floats around every half-integer of a row whose quotients fp32 cannot separate
    big1 = torch.tensor(1.0000001, device=dev)
    half = ((torch.arange(-127, 127, device=dev).double() + 0.5) * big1.double() / 127).float()
    near = torch.cat([half, torch.nextafter(half, half + 1), torch.nextafter(half, half - 1), big1[None]])[None]
    assert torch.equal(quant.quantize_rows(near)[0], _q_ref(near)[0])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k", [24, 777, 4096, 20000])
def test_rows_that_are_not_finite(cuda_device, k, dtype):
    x = _x(5, k, dtype, k, cuda_device)
    x[1, k // 2] = float("inf")
    x[2, 0] = float("nan")
    x[3] = 0
    w = torch.ones(k, device=cuda_device)
    for q, scale in (quant.quantize_rows(x), norm.rms_norm_int8(x, w)[:2]):
        assert bool(torch.isnan(scale[1:3]).all()) and int(q[1:3].abs().max()) == 0
        assert float(scale[3]) == 0 and int(q[3].abs().max()) == 0
        assert bool(torch.isfinite(scale[[0, 3, 4]]).all()) and int(q[[0, 4]].abs().amax(1).min()) == 127


def _check_norm(x, w, res, out, m, k):
    q, scale, h, rstd = out
    want_h = x if res is None else (x.float() + res.float()).to(x.dtype)
    assert torch.equal(h, want_h)
    hd = want_h.double()
    a = (want_h.float() * w)  # the definition's one fp32 product
    ref, big = _q_ref(a)
    assert torch.equal(q, ref)
    r = 1 / torch.sqrt((hd * hd).mean(1) + EPS)
    adds = 26 + k // 1024
    # the sum's relative error halves under the root; division, addition, root, reciprocal round once each
    assert bool(((rstd.double() - r).abs() <= (adds / 2 + 4) * u * r).all())
    s = big * r / 127
    assert bool(((scale.double() - s).abs() <= (adds / 2 + 7) * u * s).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,k", SIZES)
def test_rms_norm_int8(cuda_device, m, k, residual, dtype):
    dev = cuda_device
    x = _x(m, k, dtype, 7 * m + k, dev)
    res = _x(m, k, dtype, 11 * m + k, dev) if residual else None
    w = torch.randn(k, generator=_gen(dev, k), device=dev)
    if m > 2:
        x[1] = 0
        if residual:
            res[1] = 0
    out = norm.rms_norm_int8(x, w, EPS, residual=res)
    _check_norm(x, w, res, out, m, k)
    if not residual:
        assert out[2] is x


@pytest.mark.parametrize("k", [512, 777, 20000])
def test_rms_norm_int8_strided_rows_in_place_and_given_outputs(cuda_device, k):
    dev = cuda_device
    wide = _x(6, 2 * k + 24, BF16, k, dev)
    x, res = wide[:, 8:8 + k], _x(6, k + 3, BF16, k + 1, dev)[:, 3:]
    w = torch.randn(k, generator=_gen(dev, k), device=dev)
    # rows off the 16-byte grid are read one element at a time: rstd's sum runs in another order,
    # so each layout is held to the definition rather than to another layout's bits
    _check_norm(x, w, res, norm.rms_norm_int8(x, w, EPS, residual=res), 6, k)
    buf = torch.full((8, k + 5), 77, dtype=torch.int8, device=dev)
    q = buf[1:7, 2:2 + k]
    scale, rstd = torch.empty(6, device=dev), torch.empty(6, device=dev)
    stream = res.clone()
    out = norm.rms_norm_int8(x, w, EPS, residual=stream, q=q, scale=scale, rstd=rstd, h=stream)
    assert out[0] is q and out[1] is scale and out[2] is stream and out[3] is rstd
    _check_norm(x, w, res, out, 6, k)
    buf[1:7, 2:2 + k] = 77
    assert bool((buf == 77).all())  # nothing beside the rows was written


def _bwd_ref(dy, h, w, rstd, dh):
    dy, h, w, r = dy.double(), h.double(), w.double(), rstd.double()[:, None]
    xh, g = h * r, dy * w
    dx = r * (g - xh * (g * xh).mean(1, keepdim=True))
    size = r * (g.abs() + xh.abs() * (g * xh).abs().mean(1, keepdim=True))
    if dh is not None:
        dx = dx + dh.double()
        size = size + dh.double().abs()
    return dx, size, (dy * xh).sum(0), (dy * xh).abs().sum(0)


def _bwd_inputs(m, k, dtype, dh, dev, seed):
    h = _x(m, k, dtype, seed, dev)
    g = _gen(dev, seed + 1)
    dy = torch.randn((m, k), generator=g, device=dev).to(dtype)
    w = torch.randn(k, generator=g, device=dev)
    d = torch.randn((m, k), generator=g, device=dev).to(dtype) if dh else None
    rstd = torch.rsqrt(h.float().square().mean(1) + EPS)
    return dy, h, w, rstd, d


def _check_bwd(dy, h, w, rstd, d, dx, dw):
    m, k = h.shape
    rx, size, rw, rsize = _bwd_ref(dy, h, w, rstd, d)
    half = 2.0 ** -8 if h.dtype == BF16 else u
    # fp32 steps: the row's mean (26 + K / 1024 additions, products), then four roundings
    tol = half * rx.abs() + (34 + k // 1024) * u * size
    assert bool(((dx.double() - rx).abs() <= tol).all())
    # dweight: rows of a block in sequence (or of a strip's warp), then the blocks
    assert bool(((dw.double() - rw).abs() <= (m / 64 + 128) * u * rsize).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dh", [False, True])
@pytest.mark.parametrize("m,k", SIZES + [(3000, 96), (1200, 1001), (2500, 4096), (700, 12289)])
def test_rms_norm_backward(cuda_device, m, k, dh, dtype):
    a = _bwd_inputs(m, k, dtype, dh, cuda_device, 3 * m + k)
    dx, dw = norm.rms_norm_backward(*a[:4], dh=a[4])
    _check_bwd(*a, dx, dw)
    dx2, dw2 = norm.rms_norm_backward(*a[:4], dh=a[4])
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


@pytest.mark.parametrize("k", [512, 1001, 13000])
def test_rms_norm_backward_strided_and_in_place(cuda_device, k):
    dev = cuda_device
    dy, h, w, rstd, d = _bwd_inputs(37, k, BF16, True, dev, k)
    want = norm.rms_norm_backward(dy, h, w, rstd, dh=d)
    wide = [torch.zeros((37, k + 11), dtype=BF16, device=dev) for _ in range(3)]
    views = [b[:, 5:5 + k] for b in wide]
    for v, t in zip(views, (dy, h, d)):
        v.copy_(t)
    _check_bwd(dy, h, w, rstd, d, *norm.rms_norm_backward(views[0], views[1], w, rstd, dh=views[2]))
    for out in (0, 1, 2):  # over dy, h, dh
        t = [dy.clone(), h.clone(), d.clone()]
        dx, dw = norm.rms_norm_backward(t[0], t[1], w, rstd, dh=t[2], dx=t[out])
        assert dx is t[out] and torch.equal(dx, want[0]) and torch.equal(dw, want[1])


def test_rms_norm_backward_against_differences(cuda_device):
    """Central differences in fp64 of sum(dy * y) + sum(dh * h), y the norm without its rounding."""
    dev = cuda_device
    m, k = 3, 40
    dy, h, w, _, d = _bwd_inputs(m, k, F32, True, dev, 5)
    dyd, wd, dd = dy.double(), w.double(), d.double()

    def f(hh, ww):
        r = 1 / torch.sqrt((hh * hh).mean(1, keepdim=True) + EPS)
        return float((dyd * hh * r * ww).sum() + (dd * hh).sum())

    hd = h.double()
    rstd = (1 / torch.sqrt((hd * hd).mean(1) + EPS)).float()
    dx, dw = norm.rms_norm_backward(dy, h, w, rstd, dh=d)
    step = 1e-5
    # differences: truncation step^2 times a third derivative of order |dy| / h^2, rounding 1e-15 / step
    for i in range(m):
        for j in range(0, k, 7):
            e = torch.zeros_like(hd)
            e[i, j] = step
            assert abs((f(hd + e, wd) - f(hd - e, wd)) / (2 * step) - float(dx[i, j])) <= 1e-4
    for j in range(0, k, 3):
        e = torch.zeros_like(wd)
        e[j] = step
        assert abs((f(hd, wd + e) - f(hd, wd - e)) / (2 * step) - float(dw[j])) <= 1e-4


def test_no_rows(cuda_device):
    dev = cuda_device
    x = torch.empty((0, 64), dtype=BF16, device=dev)
    w = torch.ones(64, device=dev)
    q, scale = quant.quantize_rows(x)
    assert q.shape == (0, 64) and scale.shape == (0,)
    q, scale, h, rstd = norm.rms_norm_int8(x, w, residual=x)
    assert q.shape == (0, 64) and h.shape == (0, 64)
    dw = torch.full((64,), float("nan"), device=dev)
    dx, dw = norm.rms_norm_backward(x, x, w, rstd, dweight=dw)
    assert dx.shape == (0, 64) and bool((dw == 0).all())
