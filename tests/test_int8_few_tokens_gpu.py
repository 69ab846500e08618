"""The int8 Linear forward for a token or a few: bit for bit the definition, at row ends inside a
16-byte unit with other values behind them, at every end of a mask word, and in a replayed graph."""
import pytest
import torch

from c3_b200 import _lib, linear, quant

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _rows(m, k, dev, seed):
    """int8 rows whose stride's rest is not zero, and scales."""
    g = torch.Generator(device=dev).manual_seed(seed)
    buf = torch.randint(-128, 128, (m, (k + 15) // 16 * 16), generator=g, device=dev, dtype=torch.int8)
    return buf[:, :k], torch.rand(m, generator=g, device=dev) * 0.02 + 1e-3


def _ref(xq, xs, wq, ws, b):
    z = (xq.double() @ wq.double().t()).float() * (xs[:, None] * ws[None, :])
    return z if b is None else z + b


def _bits(z):
    m, n = z.shape
    pad = torch.zeros((m, (n + 31) // 32 * 32), dtype=torch.int64, device=z.device)
    pad[:, :n] = z > 0
    words = (pad.view(m, -1, 32) << torch.arange(32, device=z.device)).sum(2)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("k", [1, 15, 16, 17, 500, 512, 513, 1024, 1030, 4095, 9000, 20000])
@pytest.mark.parametrize("n", [1, 7, 8, 31, 33, 200])
def test_few_tokens(cuda_device, m, n, k):
    dev = cuda_device
    xq, xs = _rows(m, k, dev, 1 + k)
    wq, ws = _rows(n, k, dev, 2 + n)
    b = torch.randn(n, generator=torch.Generator(device=dev).manual_seed(3), device=dev)
    z = _ref(xq, xs, wq, ws, b)
    buf = torch.full((m + 1, (n + 31) // 32 + 1), 77, dtype=torch.int32, device=dev)
    ybuf = torch.full((m + 1, n + 3), 5.0, device=dev)
    y, mask = linear.forward_int8(xq, xs, wq, ws, b, Y=ybuf[:m, 1:1 + n], mask=buf[:m, :-1], out_dtype=F32)
    assert torch.equal(y, z.clamp_min(0)) and torch.equal(mask, _bits(z))
    assert bool((buf[:m, -1] == 77).all()) and bool((buf[m] == 77).all())
    assert bool((ybuf[:, 0] == 5).all()) and bool((ybuf[:, n + 1:] == 5).all()) and bool((ybuf[m] == 5).all())
    y, mask = linear.forward_int8(xq, xs, wq, ws, None, relu=False, out_dtype=BF16)
    assert mask is None and torch.equal(y, _ref(xq, xs, wq, ws, None).to(BF16))


@pytest.mark.parametrize("m", [1, 2, 4])
@pytest.mark.parametrize("n,k", [(4096, 4096), (12288, 1024), (2400, 4096), (130, 131071)])
def test_few_tokens_many_blocks_and_long_rows(cuda_device, m, n, k):
    dev = cuda_device
    xq, xs = _rows(m, k, dev, 1)
    wq, ws = _rows(n, k, dev, 2)
    y, _ = linear.forward_int8(xq, xs, wq, ws, relu=False, out_dtype=F32)
    assert torch.equal(y, _ref(xq, xs, wq, ws, None))


def test_few_tokens_same_bits_as_many(cuda_device):
    """A token's row does not depend on how many tokens came with it."""
    dev = cuda_device
    xq, xs = _rows(300, 777, dev, 1)
    wq, ws = _rows(200, 777, dev, 2)
    b = torch.randn(200, device=dev)
    y, mask = linear.forward_int8(xq, xs, wq, ws, b, out_dtype=F32)
    for m in (1, 2, 3, 4, 16):
        ym, mm = linear.forward_int8(xq[7:7 + m], xs[7:7 + m], wq, ws, b, out_dtype=F32)
        assert torch.equal(ym, y[7:7 + m]) and torch.equal(mm, mask[7:7 + m])


def test_few_tokens_not_finite(cuda_device):
    dev = cuda_device
    xq, xs = _rows(3, 64, dev, 1)
    wq, ws = _rows(40, 64, dev, 2)
    xs[1] = float("nan")
    y, mask = linear.forward_int8(xq, xs, wq, ws)
    assert bool(torch.isnan(y[1]).all()) and bool((mask[1] == 0).all())
    assert bool(torch.isfinite(y[[0, 2]]).all())


def test_few_tokens_given_ctas(cuda_device):
    """The cap on GEMM CTAs holds here too: the persistent kernel then runs, with the same bits."""
    dev = cuda_device
    xq, xs = _rows(2, 640, dev, 1)
    wq, ws = _rows(1000, 640, dev, 2)
    y, mask = linear.forward_int8(xq, xs, wq, ws)
    _lib.load().c3cu_set_gemm_max_ctas(8)
    try:
        y8, mask8 = linear.forward_int8(xq, xs, wq, ws)
    finally:
        _lib.load().c3cu_set_gemm_max_ctas(0)
    assert torch.equal(y, y8) and torch.equal(mask, mask8)


def test_few_tokens_in_graphs_on_two_streams(cuda_device):
    """Two captured decoding steps (quantise, product) replayed at once on two streams."""
    dev = cuda_device
    wq, ws = _rows(500, 1000, dev, 2)
    b = torch.randn(500, device=dev)
    runs = []
    for s in range(2):
        x = torch.zeros((1, 1000), device=dev)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            q, sc = quant.quantize_rows(x)
            y, mask = linear.forward_int8(q, sc, wq, ws, b, out_dtype=F32)
        runs.append((x, stream, graph, q, sc, y, mask))
    for step in range(3):
        for s, (x, *_rest) in enumerate(runs):
            x.copy_(torch.randn((1, 1000), generator=torch.Generator(device=dev).manual_seed(10 * step + s), device=dev))
        torch.cuda.synchronize()
        for _x, stream, graph, *_rest in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _x, _s, _g, q, sc, y, mask in runs:
            z = _ref(q, sc, wq, ws, b)
            assert torch.equal(y, z.clamp_min(0)) and torch.equal(mask, _bits(z))
