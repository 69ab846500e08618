"""The row kernels for many rows, which come through a ring of buffers in shared memory: random data in every
row, at numbers of rows just below, at and above those from which a B200 (148 SMs) takes the ring, on and off
the 16-byte grid, in place, between neighbours that must stay, and with rows that are not finite."""
import pytest
import torch

from c3_b200 import norm, quant
from tests.test_int8_rows_gpu import (BF16, EPS, F32, _bwd_inputs, _by_127, _check_bwd, _check_norm, _gen, _q_ref, _x)

pytestmark = pytest.mark.gpu


def _kernels(call):
    """Names of the kernels that a call launches, or None where the profiler sees no GPU."""
    from torch.profiler import ProfilerActivity, profile
    torch.cuda.synchronize()
    try:
        with profile(activities=[ProfilerActivity.CUDA], acc_events=True) as p:
            call()
            torch.cuda.synchronize()
    except RuntimeError:  # the profiler's, where another tool holds the GPU's counters
        return None
    names = [e.key for e in p.key_averages() if "kernel" in e.key]
    return names or None


def _spoil(x):
    """Rows that are not finite, or zero: the first and last, which off the grid are read past the ring, and one
    that a block meets later."""
    m, k = x.shape
    x[0, k - 1] = float("nan")
    x[m - 1, 0] = float("inf")
    x[m // 2 + 3] = 0
    x[m // 2, k // 2] = float("-inf")
    x[m // 3, :] = float("nan")
    return [0, m // 3, m // 2, m - 1], m // 2 + 3


# (columns, least rows of the ring, type): by the blocks an SM holds and the rows a block then has
QUANTISE = [(4096, 9472, BF16), (12288, 592, BF16), (8704, 888, F32), (777, 4736, BF16), (3100, 2368, BF16),
            (6201, 1184, BF16), (12301, 592, BF16)]
NORM = [(4096, 4736, BF16), (12288, 296, BF16), (8704, 296, F32), (777, 4736, BF16), (3100, 2368, BF16),
        (6201, 1184, BF16), (12301, 592, BF16)]


def _wide(m, k, dtype, dev, seed, at):
    """x as columns at.. of a wider buffer, and the buffer."""
    unit = 16 // torch.empty((), dtype=dtype).element_size()
    buf = torch.full((m, (k + 2 * unit) // unit * unit), 5.0, dtype=dtype, device=dev)
    v = buf[:, at:at + k]
    v.copy_(_x(m, k, dtype, seed, dev))
    return v, buf


@pytest.mark.parametrize("more", [-1, 0, 129])
@pytest.mark.parametrize("k,least,dtype", QUANTISE + [(8704, 592, F32)])
def test_quantise(cuda_device, k, least, dtype, more):
    m = least + more
    x = _x(m, k, dtype, m, cuda_device)
    q, scale = quant.quantize_rows(x)
    ref, big = _q_ref(x)
    assert torch.equal(q, ref) and torch.equal(scale, _by_127(big))
    bad, zero = _spoil(x)
    rest = torch.ones(m, dtype=torch.bool, device=cuda_device)
    rest[bad] = False
    q, scale = quant.quantize_rows(x)
    assert torch.equal(q[rest], torch.where((torch.arange(m, device=cuda_device) == zero)[:, None], 0, ref)[rest])
    assert bool(torch.isnan(scale[bad]).all()) and int(q[bad].abs().max()) == 0 and float(scale[zero]) == 0
    assert bool(torch.isfinite(scale[rest]).all())


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("more", [-1, 0, 129])
@pytest.mark.parametrize("k,least,dtype", NORM)
def test_norm(cuda_device, k, least, dtype, more, residual):
    m, dev = least + more, cuda_device
    x = _x(m, k, dtype, m, dev)
    res = _x(m, k, dtype, m + 1, dev) if residual else None
    w = torch.randn(k, generator=_gen(dev, k), device=dev)
    out = norm.rms_norm_int8(x, w, EPS, residual=res)
    _check_norm(x, w, res, out, m, k)
    bad, zero = _spoil(x)
    if residual:
        res[zero] = 0
    q, scale, h, rstd = norm.rms_norm_int8(x, w, EPS, residual=res)
    rest = torch.ones(m, dtype=torch.bool, device=dev)
    rest[bad] = False
    assert bool(torch.isnan(scale[bad]).all()) and int(q[bad].abs().max()) == 0
    _check_norm(x[rest], w, res[rest] if residual else None, (q[rest], scale[rest], h[rest], rstd[rest]), m, k)
    assert float(scale[zero]) == 0 and int(q[zero].abs().max()) == 0


@pytest.mark.parametrize("k,m,dtype", [(4096, 4801, BF16), (4095, 2401, BF16), (777, 4801, BF16), (6199, 1211, BF16),
                                       (12288, 301, BF16), (12287, 611, BF16), (8704, 301, F32)])
def test_norm_between_neighbours_and_in_place(cuda_device, k, m, dtype):
    """x and the residual at different columns of wider buffers, so that their rows start at different places
    of a 16-byte piece; then the sum over either of them."""
    dev = cuda_device
    x, xbuf = _wide(m, k, dtype, dev, 1, 0 if k % 8 == 0 else 3)
    res, rbuf = _wide(m, k, dtype, dev, 2, 0 if k % 8 == 0 else 6)
    w = torch.randn(k, generator=_gen(dev, k), device=dev)
    keep, rkeep = x.clone(), res.clone()
    qbuf = torch.full((m + 2, k + 7), 77, dtype=torch.int8, device=dev)
    q = qbuf[1:m + 1, 5:5 + k]
    out = norm.rms_norm_int8(x, w, EPS, residual=res, q=q)
    _check_norm(keep, w, rkeep, out, m, k)
    qbuf[1:m + 1, 5:5 + k] = 77
    assert bool((qbuf == 77).all())
    out = norm.rms_norm_int8(x, w, EPS, residual=res, h=res)
    assert out[2] is res
    _check_norm(keep, w, rkeep, out, m, k)
    res.copy_(rkeep)
    out = norm.rms_norm_int8(x, w, EPS, residual=res, h=x)
    assert out[2] is x
    _check_norm(keep, w, rkeep, out, m, k)
    for v, buf in ((x, xbuf), (res, rbuf)):
        v.fill_(5.0)
        assert bool((buf == 5.0).all())


@pytest.mark.parametrize("m,k", [(2500, 4096), (2500, 4095), (6000, 100), (1500, 1001), (700, 12288), (700, 12287)])
def test_gradient_in_place(cuda_device, m, k):
    """dx over dy, over h and over dh has the bits of dx elsewhere."""
    dev = cuda_device
    dy, h, w, rstd, d = _bwd_inputs(m, k, BF16, True, dev, k)
    want = norm.rms_norm_backward(dy, h, w, rstd, dh=d)
    _check_bwd(dy, h, w, rstd, d, *want)
    for out in range(3):
        t = [dy.clone(), h.clone(), d.clone()]
        dx, dw = norm.rms_norm_backward(t[0], t[1], w, rstd, dh=t[2], dx=t[out])
        assert dx is t[out] and torch.equal(dx, want[0]) and torch.equal(dw, want[1])


def test_these_sizes_take_the_ring(cuda_device):
    dev = cuda_device
    if torch.cuda.get_device_properties(dev).multi_processor_count != 148:
        pytest.skip("the thresholds above are those of 148 SMs")
    for k, least, dtype in QUANTISE:
        for m, ring in ((least - 1, False), (least, True)):
            x = _x(m, k, dtype, 1, dev)
            names = _kernels(lambda: quant.quantize_rows(x))
            if names is None:
                pytest.skip("no kernel names here")
            assert any("ring_rows_kernel" in n for n in names) is ring, (m, k, names)
    for k, least, dtype in NORM:
        w = torch.ones(k, device=dev)
        for m, ring in ((least - 1, False), (least, True)):
            x = _x(m, k, dtype, 1, dev)
            for res in (None, x):
                names = _kernels(lambda: norm.rms_norm_int8(x, w, residual=res))
                assert any("ring_rows_kernel" in n for n in names) is ring, (m, k, names)
