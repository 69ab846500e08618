"""Given outputs of the 8-bit path that share memory with an input or with another output are refused
before any C call; other columns of one buffer are not shared memory."""
import random

import pytest
import torch

from c3_b200 import linear, norm, quant
from tests.test_int8_checks_cpu import any_device, bf16, f32, i8, i32, no_library, refused, z  # noqa: F401

M, N, K = 8, 64, 32


def passes(fn, *args, **kwargs):
    """Gets past the checks, to the device or the library, which are not there."""
    with pytest.raises((AssertionError, AttributeError, RuntimeError)) as e:
        fn(*args, **kwargs)
    assert "overlaps" not in str(e.value)


def test_overlap_against_every_byte():
    rng = random.Random(1)
    pool = torch.zeros(4096, dtype=torch.uint8)

    def view():
        kind = rng.choice((i8, bf16, f32))
        size = torch.empty((), dtype=kind).element_size()
        base = pool[rng.randrange(0, 256, 4):]
        base = base[:base.numel() // 4 * 4].view(kind)
        if rng.random() < 0.3:
            return base[:rng.randrange(0, 40)]
        rows, cols = rng.randrange(1, 6), rng.randrange(1, 12)
        return base.as_strided((rows, cols), (rng.choice((16, 32, 64)) // size if 16 // size >= cols else cols + 16, 1))

    def bytes_of(t):
        a, rows, ld, width = linear._rows_span(t)
        return {a + r * ld + i for r in range(rows) for i in range(width)}
    shared = 0
    for _ in range(4000):
        p, q = view(), view()
        really = bool(bytes_of(p) & bytes_of(q))
        told = linear._overlap(p, q)
        shared += really
        assert told or not really
        (_, m, lda, _), (_, n, ldb, _) = linear._rows_span(p), linear._rows_span(q)
        if told and not really:  # only rows of different strides may be told so, or a row between others
            assert m > 1 and n > 1 and lda != ldb or 1 in (m, n)
    assert 500 < shared < 3500


def test_quantize_rows(any_device):  # noqa: F811
    x = z(M, K, dtype=f32)
    refused(quant.quantize_rows, x, scale=x.view(-1)[:M], match="overlaps x")
    q = z(M, K, dtype=i8)
    refused(quant.quantize_rows, x, q=q, scale=q.view(-1)[:4 * M].view(f32), match="overlaps q")
    both = z(M, 2 * K, dtype=i8)
    passes(quant.quantize_rows, z(M, K), q=both[:, :K])


def test_rms_norm(any_device):  # noqa: F811
    x, r, w = z(M, K, dtype=f32), z(M, K, dtype=f32), z(K, dtype=f32)
    for given in ("scale", "rstd"):
        for t, other in ((x, "x"), (r, "residual"), (w, "weight")):
            refused(norm.rms_norm_int8, x, w, residual=r, **{given: t.view(-1)[:M]}, match=f"overlaps {other}")
    v = z(M, dtype=f32)
    refused(norm.rms_norm_int8, x, w, scale=v, rstd=v, match="overlaps scale")
    q = z(M, K, dtype=i8)
    refused(norm.rms_norm_int8, x, w, q=q, rstd=q.view(-1)[:4 * M].view(f32), match="overlaps q")
    flat = z(M * K + K, dtype=f32)
    refused(norm.rms_norm_int8, x, flat[M * K - 4:M * K - 4 + K], residual=r, h=flat[:M * K].view(M, K),
            match="overlaps weight")
    passes(norm.rms_norm_int8, x, w, residual=r, h=r, q=q, scale=v, rstd=z(M, dtype=f32))


def test_rms_norm_backward(any_device):  # noqa: F811
    dy, h, dh, w, r = z(M, K, dtype=f32), z(M, K, dtype=f32), z(M, K, dtype=f32), z(K, dtype=f32), z(M, dtype=f32)
    for t, other in ((dy, "dy"), (h, "h"), (dh, "dh"), (w, "weight")):
        refused(norm.rms_norm_backward, dy, h, w, r, dh=dh, dweight=t.view(-1)[:K], match=f"overlaps {other}")
    long = z(K + M, dtype=f32)
    refused(norm.rms_norm_backward, dy, h, w, long[K - 1:K - 1 + M], dweight=long[:K], match="overlaps rstd")
    dx = z(M, K, dtype=f32)
    refused(norm.rms_norm_backward, dy, h, w, r, dx=dx, dweight=dx[1], match="overlaps dx")
    flat = z(M * K + K, dtype=f32)
    refused(norm.rms_norm_backward, dy, h, flat[M * K - 4:M * K - 4 + K], r, dx=flat[:M * K].view(M, K),
            match="overlaps weight")
    for out in (dy, h, dh, dx):
        passes(norm.rms_norm_backward, dy, h, w, r, dh=dh, dx=out, dweight=z(K, dtype=f32))


def test_forward_int8(any_device):  # noqa: F811
    words = (N + 31) // 32
    xq, xs, wq, ws, b = z(M, K, dtype=i8), z(M, dtype=f32), z(N, K, dtype=i8), z(N, dtype=f32), z(N, dtype=f32)
    for t, other in ((wq, "Wq"), (xq, "Xq")):
        refused(linear.forward_int8, xq, xs, wq, ws, b, mask=t.view(-1)[:4 * M * words].view(i32).view(M, words),
                match=f"overlaps {other}")
    big = z(M * N, dtype=f32)
    refused(linear.forward_int8, xq, big[5:5 + M], wq, ws, b, out_dtype=f32, Y=big.view(M, N), match="overlaps x_scale")
    refused(linear.forward_int8, xq, xs, wq, big[5:5 + N], b, Y=big.view(M, N), match="overlaps w_scale")
    refused(linear.forward_int8, xq, xs, wq, ws, big[5:5 + N], Y=big.view(M, N), match="overlaps b")
    refused(linear.forward_int8, xq, xs, wq, ws, b, Y=big.view(M, N), mask=big.view(i32).view(M, N)[:, 7:7 + words],
            match="overlaps Y")
    wide = z(M, N + words, dtype=f32)  # the mask beside Y in one buffer
    passes(linear.forward_int8, xq, xs, wq, ws, b, Y=wide[:, :N], mask=wide.view(i32)[:, N:])


def test_grad_weight_int8(any_device):  # noqa: F811
    dz, xq = z(M, N), z(M, K, dtype=i8)
    flat = z(N * K)
    refused(linear.grad_weight_int8, dz, xq, flat.view(f32)[:M], dW=flat.view(N, K), match="overlaps x_scale")
    buf = z(N, K + N)
    refused(linear.grad_weight_int8, buf[:M, :N], xq, z(M, dtype=f32), dW=buf[:, 4:4 + K], match="overlaps dZ")
    passes(linear.grad_weight_int8, buf[:M, :N], xq, z(M, dtype=f32), dW=buf[:, N:])
