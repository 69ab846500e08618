"""RMS norm with the residual's addition and an int8 output, and its gradient.

Forward: h = x + residual, y = h * rstd * weight with rstd = 1 / sqrt(mean(h^2) + eps), and y
leaves as int8 rows with a scale each (see quant.py), ready for linear.forward_int8 and, kept,
for linear.grad_weight_int8. Backward: the rounding to int8 counts as the identity (a
straight-through gradient). The reference has no counterpart."""
from __future__ import annotations

import math

import torch

from . import _lib
from .linear import _ld, _p, _require, _require_rows, _stream
from .quant import _dtype_code, empty_rows


@_lib.on_tensor_device
def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
                  q: torch.Tensor | None = None, scale: torch.Tensor | None = None, h: torch.Tensor | None = None,
                  rstd: torch.Tensor | None = None):
    """(q int8 [M, K], scale fp32 [M], h [M, K], rstd fp32 [M]) of x [M, K] (bf16 or fp32).

    weight: fp32 [K]. With a residual (x's shape and type), h = x + residual rounded to x's type is
    the new residual stream; it may be written over either (h=residual or h=x). Without one, h is x.
    h and rstd are what `rms_norm_backward` needs. Rows may be slices of wider ones (unit column
    stride). A row of h with an infinity or a NaN gets q = 0 and scale NaN."""
    code = _dtype_code(x, "x")
    M, K = x.shape
    if K < 1:
        raise _lib.C3CUError(-1, "x", "rows need at least one element")
    _require_rows(x, "x", x.dtype, M, K)
    _require(weight, "weight", torch.float32, 1, (K,))
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise _lib.C3CUError(-1, "eps", f"expected a finite eps >= 0, got {eps}")
    if residual is None:
        if h is not None:
            raise _lib.C3CUError(-1, "h", "without a residual h is x itself")
    else:
        _require_rows(residual, "residual", x.dtype, M, K)
        if h is None:
            h = torch.empty(M, K, dtype=x.dtype, device=x.device)
        else:
            _require_rows(h, "h", x.dtype, M, K)
            _require_same_rows_or_apart(h, "h", ((x, "x"), (residual, "residual")))
    if q is None:
        q = empty_rows(M, K, x.device)
    else:
        _require_rows(q, "q", torch.int8, M, K)
    if scale is None:
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
    else:
        _require(scale, "scale", torch.float32, 1, (M,))
    if rstd is None:
        rstd = torch.empty(M, dtype=torch.float32, device=x.device)
    else:
        _require(rstd, "rstd", torch.float32, 1, (M,))
    has = residual is not None
    rc = _lib.load().c3cu_rms_norm_int8(_p(x), _ld(x), _p(residual), _ld(residual) if has else 0, code, _p(weight), eps,
                                        _p(h), _ld(h) if has else 0, _p(q), _ld(q), _p(scale), _p(rstd), M, K,
                                        _stream(x.device))
    _lib.check(rc, "c3cu_rms_norm_int8")
    return q, scale, h if has else x, rstd


def _require_same_rows_or_apart(out: torch.Tensor, name: str, inputs) -> None:
    """An output may be an input's own rows (each element is read before it is written, by the same
    thread), but may not overlap one in any other way."""
    if out.numel() == 0:
        return
    for t, other in inputs:
        if t is None or (t.data_ptr() == out.data_ptr() and _ld(t) == _ld(out)):
            continue
        a, b = out.data_ptr(), t.data_ptr()
        ea = a + ((out.shape[0] - 1) * out.stride(0) + out.shape[1]) * out.element_size()
        eb = b + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size()
        if a < eb and b < ea and not _disjoint_columns(out, t):
            raise _lib.C3CUError(-1, name, f"overlaps {other} without being the same rows")


def _disjoint_columns(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices of one row stride are different columns of one buffer."""
    if a.shape[0] <= 1 or a.stride(0) != b.stride(0) or a.element_size() != b.element_size():
        return False
    ld = a.stride(0) * a.element_size()
    off = (b.data_ptr() - a.data_ptr()) % ld
    width = a.shape[1] * a.element_size()
    return off >= width and off + b.shape[1] * b.element_size() <= ld


@_lib.on_tensor_device
def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                      dh: torch.Tensor | None = None, dx: torch.Tensor | None = None,
                      dweight: torch.Tensor | None = None):
    """(dx [M, K], dweight fp32 [K]) of the norm whose forward saved h and rstd.

    dy: gradient of the normalised output; dh: gradient that reaches h past the norm (the residual
    stream's), added to dx. dx is the gradient of x and of the residual alike. dy, h, dh and dx have
    one type (bf16 or fp32); dx may be written over any of them. dweight has the same bits in every
    run."""
    code = _dtype_code(h, "h")
    M, K = h.shape
    if K < 1:
        raise _lib.C3CUError(-1, "h", "rows need at least one element")
    _require_rows(h, "h", h.dtype, M, K)
    _require_rows(dy, "dy", h.dtype, M, K)
    if dh is not None:
        _require_rows(dh, "dh", h.dtype, M, K)
    _require(weight, "weight", torch.float32, 1, (K,))
    _require(rstd, "rstd", torch.float32, 1, (M,))
    if dx is None:
        dx = torch.empty(M, K, dtype=h.dtype, device=h.device)
    else:
        _require_rows(dx, "dx", h.dtype, M, K)
        _require_same_rows_or_apart(dx, "dx", ((dy, "dy"), (h, "h"), (dh, "dh")))
    if dweight is None:
        dweight = torch.empty(K, dtype=torch.float32, device=h.device)
    else:
        _require(dweight, "dweight", torch.float32, 1, (K,))
    L = _lib.load()
    nb = L.c3cu_rms_norm_bwd_workspace(M, K)
    # of this call alone: a graph that captures it keeps its own
    ws = torch.empty(nb, dtype=torch.uint8, device=h.device) if nb else None
    rc = L.c3cu_rms_norm_bwd(_p(dy), _ld(dy), _p(h), _ld(h), _p(dh), _ld(dh) if dh is not None else 0, code, _p(weight),
                             _p(rstd), _p(dx), _ld(dx), _p(dweight), M, K, _p(ws), nb, _stream(h.device))
    _lib.check(rc, "c3cu_rms_norm_bwd")
    return dx, dweight
