"""The int8 Linear forward and the weight gradient from an 8-bit checkpoint, against plain
computations, and the whole path as a training step uses it.

The forward is compared bit for bit: its integer sums are exact and its fp32 operations are
defined one by one."""
import pytest
import torch

import c3_b200
from c3_b200 import _lib, linear, norm, quant

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
u = 2.0 ** -24


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _rows(m, k, dev, seed):
    """Random int8 rows over the whole range (-128 too) in the 16-byte layout, and scales."""
    g = _gen(dev, seed)
    q = quant.empty_rows(m, k, dev)
    q.copy_(torch.randint(-128, 128, (m, k), generator=g, device=dev, dtype=torch.int8))
    return q, torch.rand(m, generator=g, device=dev) * 0.02 + 1e-3


def _forward_ref(xq, xs, wq, ws, b, relu):
    acc = (xq.double() @ wq.double().t()).float()  # sums below 2^53: exact, then one rounding
    z = acc * (xs[:, None] * ws[None, :])
    if b is not None:
        z = z + b
    bits = z > 0
    return (z.clamp_min(0) if relu else z), bits


def _unpack(mask, n):
    bits = (mask[:, :, None] >> torch.arange(32, device=mask.device)) & 1
    return bits.reshape(mask.shape[0], -1)[:, :n].bool(), bits.reshape(mask.shape[0], -1)[:, n:]


def _check_forward(m, n, k, dev, relu, bias, out_dtype, seed=0):
    xq, xs = _rows(m, k, dev, seed + 1)
    wq, ws = _rows(n, k, dev, seed + 2)
    b = torch.randn(n, generator=_gen(dev, seed + 3), device=dev) if bias else None
    y, mask = linear.forward_int8(xq, xs, wq, ws, b, relu=relu, out_dtype=out_dtype)
    ref, bits = _forward_ref(xq, xs, wq, ws, b, relu)
    same = torch.equal(y, ref.to(out_dtype))
    assert y.dtype == out_dtype and same, (m, n, k)
    if relu:
        got, beyond = _unpack(mask, n)
        assert torch.equal(got, bits) and not bool(beyond.any())
    else:
        assert mask is None


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 100, 128, 129, 200, 256, 257, 300, 520, 1000])
@pytest.mark.parametrize("n,k", [(16, 16), (1, 1), (100, 130), (128, 128), (300, 4096), (1397, 777), (515, 1032)])
def test_forward_int8_sizes(cuda_device, m, n, k):
    for relu, bias, dt in ((True, True, BF16), (False, False, F32)):
        _check_forward(m, n, k, cuda_device, relu, bias, dt, seed=m + n + k)


@pytest.mark.parametrize("relu", [True, False])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(8, 256, 512), (384, 640, 320)])
def test_forward_int8_epilogues(cuda_device, m, n, k, relu, bias, out_dtype):
    _check_forward(m, n, k, cuda_device, relu, bias, out_dtype)


def test_forward_int8_large_and_long(cuda_device):
    _check_forward(4096, 4096, 4096, cuda_device, True, True, BF16)
    _check_forward(2, 130, 131071, cuda_device, False, True, F32)
    _check_forward(300, 300, 131071, cuda_device, False, True, F32)


@pytest.mark.parametrize("m", [2, 300])
def test_forward_int8_largest_sums_do_not_overflow(cuda_device, m):
    """-128 * -128 * 131071 is the largest sum the limit on K admits: 2^31 - 16384."""
    dev = cuda_device
    k = linear.INT8_MAX_K
    xq, wq = quant.empty_rows(m, k, dev), quant.empty_rows(4, k, dev)
    xq.fill_(-128)
    wq.fill_(-128)
    wq[1] = 127
    one = torch.ones(m, device=dev)
    y, _ = linear.forward_int8(xq, one, wq, one[:4] if m >= 4 else torch.ones(4, device=dev), relu=False, out_dtype=F32)
    want = torch.tensor([2 ** 14 * k, -128 * 127 * k, 2 ** 14 * k, 2 ** 14 * k], dtype=torch.float64, device=dev).float()
    assert torch.equal(y, want.expand(m, 4))


@pytest.mark.parametrize("m", [5, 300])
def test_forward_int8_slices_given_outputs_and_untouched_neighbours(cuda_device, m):
    dev = cuda_device
    n, k = 200, 208
    xw, xs = _rows(m, 512, dev, 1)
    ww, ws = _rows(n, 512, dev, 2)
    xq, wq = xw[:, 16:16 + k], ww[:, 64:64 + k]
    b = torch.randn(n, generator=_gen(dev, 3), device=dev)
    want, wmask = linear.forward_int8(xq.contiguous(), xs, wq.contiguous(), ws, b)
    ybuf = torch.full((m, n + 24), 5.0, dtype=BF16, device=dev)
    mbuf = torch.full((m, 9), -7, dtype=torch.int32, device=dev)
    y, mask = linear.forward_int8(xq, xs, wq, ws, b, Y=ybuf[:, 8:8 + n], mask=mbuf[:, 1:8])
    assert torch.equal(y, want) and torch.equal(mask, wmask)
    assert bool((ybuf[:, :8] == 5).all()) and bool((ybuf[:, 8 + n:] == 5).all())
    assert bool((mbuf[:, 0] == -7).all()) and bool((mbuf[:, 8] == -7).all())


def test_forward_int8_rows_that_are_not_finite_stay_nan(cuda_device):
    dev = cuda_device
    for m in (4, 300):
        xq, xs = _rows(m, 64, dev, 1)
        wq, ws = _rows(40, 64, dev, 2)
        xq[1] = 0
        xs[1] = float("nan")
        y, mask = linear.forward_int8(xq, xs, wq, ws, torch.zeros(40, device=dev))
        assert bool(torch.isnan(y[1]).all()) and bool((mask[1] == 0).all())
        assert bool(torch.isfinite(y[0]).all()) and bool(torch.isfinite(y[2:]).all())


def test_forward_int8_empty(cuda_device):
    dev = cuda_device
    xq, xs = _rows(0, 64, dev, 1)
    wq, ws = _rows(40, 64, dev, 2)
    y, mask = linear.forward_int8(xq, xs, wq, ws)
    assert y.shape == (0, 40) and mask.shape == (0, 2)


# ------------------------------------------------------------------ dW from a checkpoint
def _dw_exact(m, n, k, dev, seed):
    """Operands whose products and sums are exact in bf16 x bf16 -> fp32: only the output rounds."""
    g = _gen(dev, seed)
    dz = torch.randint(-2, 3, (m, n), generator=g, device=dev).to(BF16)
    q = quant.empty_rows(m, k, dev)
    q.copy_(torch.randint(-128, 128, (m, k), generator=g, device=dev, dtype=torch.int8))
    s = 2.0 ** torch.randint(-3, 1, (m,), generator=g, device=dev).float()
    return dz, q, s, (dz.double().t() @ (q.double() * s.double()[:, None])).to(F32).to(BF16)


@pytest.mark.parametrize("m", [1, 2, 63, 64, 65, 128, 500, 2048])
@pytest.mark.parametrize("n,k", [(8, 1), (16, 16), (88, 130), (256, 784), (264, 257), (1024, 777)])
def test_grad_weight_int8_exact(cuda_device, m, n, k):
    dz, q, s, want = _dw_exact(m, n, k, cuda_device, m + n + k)
    assert torch.equal(linear.grad_weight_int8(dz, q, s), want)


def test_grad_weight_int8_many_tiles_and_cut_tail(cuda_device):
    """More tiles than SM pairs, with a rest that is cut along the sum; and whole waves only."""
    for n, k, m in ((4096, 2048, 4096), (2560, 2048, 640), (4096, 4096, 8192)):
        dz, q, s, want = _dw_exact(m, n, k, cuda_device, n)
        assert torch.equal(linear.grad_weight_int8(dz, q, s), want)


@pytest.mark.parametrize("m,n,k", [(128, 256, 784), (1000, 200, 333), (4096, 512, 1024)])
def test_grad_weight_int8_real_values(cuda_device, m, n, k):
    dev = cuda_device
    x = torch.randn((m, k), generator=_gen(dev, 1), device=dev).to(BF16)
    dz = (torch.randn((m, n), generator=_gen(dev, 2), device=dev) * 1e-3).to(BF16)
    q, s = quant.quantize_rows(x)
    dw = linear.grad_weight_int8(dz, q, s)
    xd = q.double() * s.double()[:, None]
    ref = dz.double().t() @ xd
    size = dz.double().abs().t() @ xd.abs()
    # bf16 rounding of the result and of each q * s (through fp32: + u), fp32 accumulation (truncating adds: 2 u)
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + (2 * m + 2) * u) * size
    assert bool(((dw.double() - ref).abs() <= tol).all())
    # independent roundings average out: the two contribute a few 2^-9 of the norm in all
    assert float((dw.double() - ref).norm() / ref.norm()) <= 2.0 ** -8
    # and it is the same bits every time
    assert torch.equal(dw, linear.grad_weight_int8(dz, q, s))


def test_grad_weight_int8_slices_and_given_output(cuda_device):
    dev = cuda_device
    m, n, k = 300, 96, 150
    dz, q, s, want = _dw_exact(m, n, k, dev, 3)
    dzw = torch.zeros((m, n + 40), dtype=BF16, device=dev)
    dzw[:, 16:16 + n] = dz
    qw = torch.zeros((m, 256), dtype=torch.int8, device=dev)
    qw[:, 32:32 + k] = q
    buf = torch.full((n, k + 9), 3.0, dtype=BF16, device=dev)
    dw = linear.grad_weight_int8(dzw[:, 16:16 + n], qw[:, 32:32 + k], s, dW=buf[:, 4:4 + k])
    assert torch.equal(dw, want)
    assert bool((buf[:, :4] == 3).all()) and bool((buf[:, 4 + k:] == 3).all())


def test_grad_weight_int8_no_rows_and_poisoned_row(cuda_device):
    dev = cuda_device
    dz, q, s, _ = _dw_exact(0, 16, 40, dev, 1)
    assert bool((linear.grad_weight_int8(dz, q, s) == 0).all())
    dz, q, s, want = _dw_exact(70, 16, 40, dev, 1)
    s[3], q[3] = float("nan"), 0
    assert bool(torch.isnan(linear.grad_weight_int8(dz, q, s)).all())


def test_refused_layouts(cuda_device):
    """The TMA rules: rows on 16 bytes. Refused before anything is launched."""
    dev = cuda_device
    xq, xs = _rows(20, 64, dev, 1)
    wq, ws = _rows(40, 64, dev, 2)
    odd = torch.zeros((20, 65), dtype=torch.int8, device=dev)
    for bad in (odd[:, :64], odd.view(-1)[1:1 + 64 * 20].view(20, 64)):
        with pytest.raises(c3_b200.C3CUError) as e:
            linear.forward_int8(bad, xs, wq, ws)
        assert e.value.code == -2
        with pytest.raises(c3_b200.C3CUError) as e:
            linear.grad_weight_int8(torch.zeros((20, 16), dtype=BF16, device=dev), bad, xs)
        assert e.value.code == -2
    with pytest.raises(c3_b200.C3CUError) as e:
        linear.grad_weight_int8(torch.zeros((20, 12), dtype=BF16, device=dev), xq, xs)
    assert e.value.code == -2


# ------------------------------------------------------------------ together
def test_norm_linear_and_backward_together(cuda_device):
    """A pre-norm Linear layer forward and backward on the 8-bit path, against fp64 on the same
    quantised operands, with the mask of the forward."""
    dev = cuda_device
    m, k, n = 384, 512, 640
    x = torch.randn((m, k), generator=_gen(dev, 1), device=dev).to(BF16)
    r = torch.randn((m, k), generator=_gen(dev, 2), device=dev).to(BF16)
    gamma = 1 + 0.1 * torch.randn(k, generator=_gen(dev, 3), device=dev)
    w = (torch.randn((n, k), generator=_gen(dev, 4), device=dev) * 0.02).to(BF16)
    b = torch.randn(n, generator=_gen(dev, 5), device=dev) * 0.01
    dy = (torch.randn((m, n), generator=_gen(dev, 6), device=dev) * 1e-3).to(BF16)
    dstream = (torch.randn((m, k), generator=_gen(dev, 7), device=dev) * 1e-3).to(BF16)

    wq, ws = quant.quantize_rows(w)
    q, s, h, rstd = norm.rms_norm_int8(x, gamma, residual=r)
    y, mask = linear.forward_int8(q, s, wq, ws, b)
    dz, db = linear.relu_mask_db(dy, mask)
    dw = linear.grad_weight_int8(dz, q, s)
    dn = linear.grad_input(dz, w)
    dx, dgamma = norm.rms_norm_backward(dn, h, gamma, rstd, dh=dstream)
    torch.cuda.synchronize()

    ref, bits = _forward_ref(q, s, wq, ws, b, True)
    assert torch.equal(y, ref.to(BF16))
    dz_ref = torch.where(bits, dy, torch.zeros_like(dy)).double()
    assert torch.equal(dz.double(), dz_ref)
    dw_ref = dz_ref.t() @ (q.double() * s.double()[:, None])
    assert float((dw.double() - dw_ref).norm() / dw_ref.norm()) <= 2.0 ** -8
    hd = (x.float() + r.float()).to(BF16).double()
    rd = 1 / torch.sqrt((hd * hd).mean(1, keepdim=True) + 1e-6)
    g, xh = dn.double() * gamma.double(), hd * rd
    dx_ref = rd * (g - xh * (g * xh).mean(1, keepdim=True)) + dstream.double()
    assert float((dx.double() - dx_ref).norm() / dx_ref.norm()) <= 2.0 ** -8
    dg_ref = (dn.double() * xh).sum(0)
    assert float((dgamma.double() - dg_ref).norm() / dg_ref.norm()) <= 1e-5
    # the int8 forward stands for the bf16 one: 127 steps per row amplitude
    y16, _ = linear.forward((hd * rd * gamma.double()).to(BF16), w, b)
    assert float((y.float() - y16.float()).norm() / y16.float().norm()) <= 0.03


def test_side_stream_and_graph_replay(cuda_device):
    """The path on a stream of its own, captured and replayed on new inputs, beside a second
    captured graph of the same calls."""
    dev = cuda_device
    m, k, n = 300, 512, 264
    gamma = torch.ones(k, device=dev)
    wq, ws = _rows(n, k, dev, 9)

    def path(x, dy):
        q, s, h, rstd = norm.rms_norm_int8(x, gamma, residual=x)
        y, mask = linear.forward_int8(q, s, wq, ws)
        dz, _ = linear.relu_mask_db(dy, mask)
        dw = linear.grad_weight_int8(dz, q, s)
        dx, dg = norm.rms_norm_backward(x, h, gamma, rstd)
        return y, dw, dx, dg

    def inputs(seed):
        return (torch.randn((m, k), generator=_gen(dev, seed), device=dev).to(BF16),
                torch.randn((m, n), generator=_gen(dev, seed + 50), device=dev).to(BF16))

    want = {s: [t.clone() for t in path(*inputs(s))] for s in (1, 2, 3)}
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = path(*inputs(1))
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    graphs = []
    for s in (1, 2):
        x, dy = inputs(s)
        with torch.cuda.stream(side):
            path(x, dy)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = path(x, dy)
        graphs.append((g, x, dy, out))
    for turn in ((1, 2), (3, 1), (2, 3)):
        for (g, x, dy, out), s in zip(graphs, turn):
            a, b = inputs(s)
            x.copy_(a)
            dy.copy_(b)
            g.replay()
        torch.cuda.synchronize()
        for (g, x, dy, out), s in zip(graphs, turn):
            assert all(torch.equal(a, b) for a, b in zip(out, want[s]))


def test_cap_on_ctas_changes_no_bits(cuda_device):
    """c3cu_set_gemm_max_ctas also bounds the int8 GEMMs; the forward's bits do not change, dW's
    stay within its own bound (another cut of the sum)."""
    dev = cuda_device
    L = _lib.load()
    xq, xs = _rows(600, 256, dev, 1)
    wq, ws = _rows(600, 256, dev, 2)
    dz, q, s, want = _dw_exact(700, 600, 520, dev, 3)
    y, mask = linear.forward_int8(xq, xs, wq, ws)
    try:
        L.c3cu_set_gemm_max_ctas(6)
        y2, mask2 = linear.forward_int8(xq, xs, wq, ws)
        dw2 = linear.grad_weight_int8(dz, q, s)
    finally:
        L.c3cu_set_gemm_max_ctas(0)
    assert torch.equal(y, y2) and torch.equal(mask, mask2)
    assert torch.equal(dw2, want)


@pytest.mark.parametrize("options", [{}, {"overlap_dx": True}, {"chunks": 2}])
def test_training_step_with_an_int8_checkpoint(cuda_device, options):
    """LinearReluTrainStep(x_checkpoint="int8"): forward, mask, db and dX are those of the bf16 step,
    bit for bit; dW is the product with the checkpoint, and near the bf16 step's."""
    from c3_b200.data_parallel import LinearReluTrainStep
    dev = cuda_device
    m, n, k = 512, 384, 328
    X = torch.randn((m, k), generator=_gen(dev, 1), device=dev).to(BF16)
    W = (torch.randn((n, k), generator=_gen(dev, 2), device=dev) * 0.05).to(BF16)
    b = torch.randn(n, generator=_gen(dev, 3), device=dev) * 0.05
    dY = (torch.randn((m, n), generator=_gen(dev, 4), device=dev) * 1e-3).to(BF16)
    ref = LinearReluTrainStep(m, n, k, dev, **options)
    step = LinearReluTrainStep(m, n, k, dev, x_checkpoint="int8", **options)
    ref(X, W, b, dY)
    step(X, W, b, dY)
    torch.cuda.synchronize()
    for name in ("Y", "mask", "dZ", "db", "dX"):
        assert torch.equal(getattr(step, name), getattr(ref, name)), name
    q, s = quant.quantize_rows(X)
    assert torch.equal(step.Xq, q) and torch.equal(step.x_scale, s)
    want = step.dZ.double().t() @ (q.double() * s.double()[:, None])
    assert float((step.dW.double() - want).norm() / want.norm()) <= 2.0 ** -8
    # a checkpoint's element is off by at most half a step, A / 254, that is about 3.5 / 254 of the
    # rows' standard deviation at most, uniformly: 0.8 % of the norm
    assert float((step.dW.double() - ref.dW.double()).norm() / ref.dW.double().norm()) <= 0.02
    for bad in ({"x_checkpoint": "int4"}, {"x_checkpoint": "int8", "grad_dtype": torch.float32},
                {"x_checkpoint": "int8", "collective": "fused"}):
        with pytest.raises(ValueError):
            LinearReluTrainStep(m, n, k, dev, **bad)
