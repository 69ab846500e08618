"""The weight gradient from an 8-bit checkpoint over the sizes at which its forms change: small tiles
of 32, 64 and 128 rows, whole or split over clusters of two to eight, large tiles with X widened on the
way or before."""
import pytest
import torch

from c3_b200 import linear, quant

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _rows16(m, cols, dtype, dev, fill):
    """A matrix whose rows start on 16 bytes, `fill` behind their ends."""
    unit = 16 // torch.empty((), dtype=dtype).element_size()
    buf = torch.full((m, (cols + unit - 1) // unit * unit), fill, dtype=dtype, device=dev)
    return buf[:, :cols]


def _exact_case(m, n, k, dev, seed):
    """Products and sums that are exact in bf16 x bf16 -> fp32: only the output rounds. The scales
    are powers of two and |q scale dz| <= 128 * 2, multiples of 2^-3, so sums stay below 2^24 units
    for m <= 8192 (2^8 * 2^13 * 2^3 = 2^24)."""
    g = _gen(dev, seed)
    dz = _rows16(m, n, BF16, dev, 3.0)
    dz.copy_(torch.randint(-2, 3, (m, n), generator=g, device=dev).to(BF16))
    q = _rows16(m, k, torch.int8, dev, 99)
    q.copy_(torch.randint(-128, 128, (m, k), generator=g, device=dev, dtype=torch.int8))
    s = 2.0 ** torch.randint(-3, 1, (m,), generator=g, device=dev).float()
    return dz, q, s, (dz.double().t() @ (q.double() * s.double()[:, None])).to(F32).to(BF16)


SIZES = [(1, 16, 1), (3, 24, 7021), (64, 8, 127), (65, 32, 129), (128, 256, 784), (130, 40, 4220), (147, 80, 461),
         (500, 1480, 255), (786, 208, 1045), (776, 56, 2464), (997, 56, 33), (1425, 16, 213), (2048, 1024, 1024),
         (2908, 32, 25), (4096, 512, 512), (8192, 96, 300), (8192, 200, 40), (7, 5808, 208), (128, 4096, 4096),
         (450, 2816, 224), (576, 2176, 4822), (1000, 1000, 1000), (6552, 272, 2500)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_exact_sums(cuda_device, m, n, k):
    dz, q, s, want = _exact_case(m, n, k, cuda_device, m + n + k)
    buf = torch.full((n + 1, k + 5), 7.0, dtype=BF16, device=cuda_device)
    dw = linear.grad_weight_int8(dz, q, s, dW=buf[:n, 3:3 + k])
    assert torch.equal(dw, want)
    assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 3 + k:] == 7).all()) and bool((buf[n] == 7).all())
    assert torch.equal(linear.grad_weight_int8(dz, q, s), want)


@pytest.mark.parametrize("m,n,k", [(128, 256, 784), (997, 56, 33), (776, 56, 2464), (10273, 448, 96), (2048, 1024, 1024)])
def test_real_values(cuda_device, m, n, k):
    dev = cuda_device
    x = torch.randn((m, k), generator=_gen(dev, 1), device=dev).to(BF16)
    dz = (torch.randn((m, n), generator=_gen(dev, 2), device=dev) * 1e-3).to(BF16)
    q, s = quant.quantize_rows(x)
    dw = linear.grad_weight_int8(dz, q, s)
    xd = q.double() * s.double()[:, None]
    ref = dz.double().t() @ xd
    size = dz.double().abs().t() @ xd.abs()
    # bf16 rounding of the result and of each q * s, and fp32 sums whose adds may truncate (2 * 2^-24 each)
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + (2 * m + 2) * 2.0 ** -24) * size
    assert bool(((dw.double() - ref).abs() <= tol).all())
    for _ in range(3):  # the same bits every time
        assert torch.equal(dw, linear.grad_weight_int8(dz, q, s))


@pytest.mark.parametrize("m,n,k", [(128, 64, 100), (997, 56, 33), (2048, 1024, 1024)])
def test_a_row_that_was_not_finite(cuda_device, m, n, k):
    dz, q, s, _ = _exact_case(m, n, k, cuda_device, 5)
    q[m // 2], s[m // 2] = 0, float("nan")
    assert bool(torch.isnan(linear.grad_weight_int8(dz, q, s)).all())


def test_two_graphs_at_once(cuda_device):
    """Captured calls replayed on two streams at once, a split small tile and a cut large one in each."""
    dev = cuda_device
    cases = [[_exact_case(m, n, k, dev, 10 * i + j) for j, (m, n, k) in
              enumerate(((997, 56, 33), (4096, 1024, 512), (8000, 264, 2056)))] for i in range(2)]
    graphs = []
    for case in cases:
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = [linear.grad_weight_int8(dz, q, s) for dz, q, s, _ in case]
        graphs.append((stream, graph, outs))
    for _ in range(3):
        for _stream, _graph, outs in graphs:
            for o in outs:
                o.zero_()
        torch.cuda.synchronize()
        for stream, graph, _outs in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for case, (_s, _g, outs) in zip(cases, graphs):
            for (_dz, _q, _sc, want), got in zip(case, outs):
                assert torch.equal(got, want)
