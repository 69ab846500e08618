"""Ways of calling the 8-bit path beside the plain one: through the C++ binding and through Python,
captured as a process's first call, with launches overlapped, from two threads, on odd pointers."""
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from c3_b200 import _lib, linear, norm, quant

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


class _NoFast:
    """A binding that leaves every call to the Python wrapper."""

    def __getattr__(self, name):
        return lambda *a: None


def _inputs(dev, m, k, n, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)

    def r(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)
    return dict(x=r(m, k), res=r(m, k), gamma=1 + 0.1 * r(k).float(), w=r(n, k, scale=0.05), b=r(n).float(),
                dy=r(m, k, scale=1e-2), dz=r(m, (n + 7) // 8 * 8, scale=1e-3).to(BF16)[:, :n])


def _path(t):
    q, s, h, rstd = norm.rms_norm_int8(t["x"], t["gamma"], residual=t["res"])
    q1, s1, h1, rstd1 = norm.rms_norm_int8(t["x"], t["gamma"], 1e-5)
    wq, ws = quant.quantize_rows(t["w"])
    y, mask = linear.forward_int8(q, s, wq, ws, t["b"])
    y1, none = linear.forward_int8(q1, s1, wq, ws, relu=False, out_dtype=F32)
    assert none is None and h1 is t["x"]
    dw = linear.grad_weight_int8(t["dz"], q, s)
    dx, dg = norm.rms_norm_backward(t["dy"], h, t["gamma"], rstd, dh=t["res"])
    dx1, dg1 = norm.rms_norm_backward(t["dy"], h1, t["gamma"], rstd1)
    return [q, s, h, rstd, q1, s1, rstd1, wq, ws, y, mask, y1, dw, dx, dg, dx1, dg1]


def _same(a, b):
    return all(x.shape == y.shape and x.dtype == y.dtype and torch.equal(x, y) for x, y in zip(a, b, strict=True))


SHAPES = [(1, 4096, 512), (3, 777, 40), (40, 256, 264), (333, 1416, 100), (700, 1001, 1397), (130, 9000, 72)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_both_bindings_give_the_same(cuda_device, monkeypatch, m, k, n, dtype):
    t = _inputs(cuda_device, m, k, n, dtype, m + k)
    want = _path(t)
    layout = [x.stride() for x in want]
    monkeypatch.setattr(_lib, "fast", lambda: _NoFast())
    got = _path(t)
    assert _same(got, want)
    if m > 1:  # of a single row the stride says nothing
        assert [x.stride() for x in got] == layout


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_overlapped_launches(cuda_device, dtype):
    """Each kernel waits for what it reads: chains of calls with c3cu_set_launch_overlap on have the
    bits that they have with it off."""
    dev = cuda_device
    cases = [_inputs(dev, m, k, n, dtype, 3 * i) for i, (m, k, n) in
             enumerate(SHAPES + [(2000, 1024, 1024), (512, 4096, 2048)])]
    want = [_path(t) for t in cases]
    lib = _lib.load()
    lib.c3cu_set_launch_overlap(1)
    try:
        for _ in range(3):
            got = [_path(t) for t in cases]
            torch.cuda.synchronize()
            assert all(_same(a, b) for a, b in zip(got, want))
    finally:
        lib.c3cu_set_launch_overlap(0)


def test_two_threads(cuda_device):
    dev = cuda_device
    cases = [_inputs(dev, 300, 640, 264, BF16, 1), _inputs(dev, 2, 4096, 512, F32, 2)]
    want = [_path(t) for t in cases]
    torch.cuda.synchronize()
    bad = []

    def run(t, w):
        try:
            stream = torch.cuda.Stream(dev)
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = _path(t)
                    stream.synchronize()
                    if not _same(got, w):
                        bad.append("bits")
        except Exception as e:  # seen by the test below
            bad.append(repr(e))
    threads = [threading.Thread(target=run, args=a) for a in zip(cases, want)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pointers_off_the_16_byte_grid(cuda_device, dtype):
    """The row kernels take any element's address: rows cut at an odd column give the bits of a copy
    where a row's sums are taken in the same order, and the same q and scale in any case."""
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(1)
    for m, k in ((1, 5), (70, 641), (2000, 1030), (5, 17001)):
        wide = torch.randn((m + 1, k + 9), generator=g, device=dev).to(dtype)
        x = wide[:m, 3:3 + k]
        q, s = quant.quantize_rows(x)
        q2, s2 = quant.quantize_rows(x.clone(memory_format=torch.contiguous_format))
        assert torch.equal(q, q2) and torch.equal(s, s2)


FIRST = """
import torch
from tests.test_int8_calls_gpu import _inputs, _path, _same
t = [_inputs(torch.device("cuda"), m, k, n, torch.bfloat16, 7) for m, k, n in ((2, 777, 40), (700, 1000, 1397), (2000, 1024, 512))]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = [_path(c) for c in t]
for _ in range(2):
    g.replay()
torch.cuda.synchronize()
assert all(_same(a, _path(c)) for a, c in zip(out, t))
print("captured")
"""


def test_first_calls_of_a_process_may_be_captured(cuda_device):
    r = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


def test_outputs_that_reach_into_inputs(cuda_device):
    dev = cuda_device
    x = torch.zeros((8, 64), dtype=BF16, device=dev)
    xs = torch.ones(8, device=dev)
    bytes_ = x.view(torch.int8)
    for call in (lambda: quant.quantize_rows(x, q=bytes_[:, :64]),
                 lambda: norm.rms_norm_int8(x, torch.ones(64, device=dev), q=bytes_[:, 64:]),
                 lambda: linear.forward_int8(bytes_[:, :64], xs, bytes_[:, 64:], xs, relu=False, Y=x[:, :8]),
                 lambda: linear.grad_weight_int8(x[:, :8], bytes_[:, 64:], xs, dW=x)):
        with pytest.raises(_lib.C3CUError) as e:
            call()
        assert e.value.code == -1 and "overlaps" in str(e.value)
