"""RMS norm with the residual's addition and an int8 output, and its gradient.

Forward: h = x + residual, y = h * rstd * weight with rstd = 1 / sqrt(mean(h^2) + eps), and y
leaves as int8 rows with a scale each (see quant.py), ready for linear.forward_int8 and, kept,
for linear.grad_weight_int8. Backward: the rounding to int8 counts as the identity (a
straight-through gradient). The reference has no counterpart."""
from __future__ import annotations

import math

import torch

from . import _lib
from .linear import (_call, _current_device, _fast_result, _on_gpu, _ptr, _require_apart, _rows_of,
                     _vector_of)
from .quant import _dtype_code, empty_rows, row_stride


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
                  q: torch.Tensor | None = None, scale: torch.Tensor | None = None, h: torch.Tensor | None = None,
                  rstd: torch.Tensor | None = None):
    """(q int8 [M, K], scale fp32 [M], h [M, K], rstd fp32 [M]) of x [M, K] (bf16 or fp32).

    weight: fp32 [K]. With a residual (x's shape and type), h = x + residual rounded to x's type is
    the new residual stream; it may be written over either (h=residual or h=x). Without one, h is x.
    h and rstd are what `rms_norm_backward` needs. Rows may be slices of wider ones (unit column
    stride). A row of h with an infinity or a NaN gets q = 0 and scale NaN. A row of zeros has scale 0;
    with eps = 0 (or one that is 0 in fp32) its rstd is 0 too, so that its gradients are those of a constant.
    Squares are summed in fp32: |h| up to about 1e18, beyond which rstd and scale are 0."""
    if q is None and scale is None and h is None and rstd is None and _on_gpu(x):
        r = _lib.fast().rms_norm_int8(x, weight, eps, residual)
        if r is not None:
            return _fast_result(r, "c3cu_rms_norm_int8")
    code = _dtype_code(x, "x")
    M, K = x.shape
    if K < 1:
        raise _lib.C3CUError(-1, "x", "rows need at least one element")
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise _lib.C3CUError(-1, "eps", f"expected a finite eps >= 0, got {eps}")
    dev, dtype = x.get_device(), x.dtype
    ldx = _rows_of(x, "x", dtype, M, K, dev)
    _vector_of(weight, "weight", torch.float32, K, dev)
    ldr = ldh = K
    if residual is None:
        if h is not None:
            raise _lib.C3CUError(-1, "h", "without a residual h is x itself")
    else:
        ldr = _rows_of(residual, "residual", dtype, M, K, dev)
        if h is not None:
            ldh = _rows_of(h, "h", dtype, M, K, dev)
            _require_same_rows_or_apart(h, ldh, "h", ((x, ldx, "x"), (residual, ldr, "residual")))
            _require_apart(h, "h", (weight, "weight"))
        else:
            h = torch.empty(M, K, dtype=dtype, device=x.device)
    # what a given output has to stay clear of: the inputs, h and the outputs before it
    taken = [(x, "x"), (residual, "residual"), (weight, "weight"), (h, "h")]
    if q is None:
        q, ldq = empty_rows(M, K, x.device), row_stride(K)
    else:
        ldq = _rows_of(q, "q", torch.int8, M, K, dev)
        _require_apart(q, "q", *taken)
        taken.append((q, "q"))
    if scale is None:
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
    else:
        _vector_of(scale, "scale", torch.float32, M, dev)
        _require_apart(scale, "scale", *taken)
        taken.append((scale, "scale"))
    if rstd is None:
        rstd = torch.empty(M, dtype=torch.float32, device=x.device)
    else:
        _vector_of(rstd, "rstd", torch.float32, M, dev)
        _require_apart(rstd, "rstd", *taken)
    _call("c3cu_rms_norm_int8", dev, x.data_ptr(), ldx, _ptr(residual), ldr, code, weight.data_ptr(), eps, _ptr(h), ldh,
          q.data_ptr(), ldq, scale.data_ptr(), rstd.data_ptr(), M, K)
    return q, scale, x if h is None else h, rstd


def _require_same_rows_or_apart(out: torch.Tensor, ld: int, name: str, inputs) -> None:
    """An output may be an input's own rows (each element is read before it is written, by the same
    thread) or other columns of the same buffer, but may not overlap one in any other way. All have
    one shape and type; `ld` and the inputs' middle entries are row strides."""
    rows, cols = out.shape
    if rows == 0:
        return
    size = out.element_size()
    a, width = out.data_ptr(), cols * size
    for t, ldt, other in inputs:
        if t is None:
            continue
        b = t.data_ptr()
        if a == b and (ld == ldt or rows == 1):
            continue
        if a < b + ((rows - 1) * ldt + cols) * size and b < a + ((rows - 1) * ld + cols) * size:
            off = (b - a) % (ld * size)
            if rows == 1 or ld != ldt or off < width or off + width > ld * size:
                raise _lib.C3CUError(-1, name, f"overlaps {other} without being the same rows")


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                      dh: torch.Tensor | None = None, dx: torch.Tensor | None = None,
                      dweight: torch.Tensor | None = None):
    """(dx [M, K], dweight fp32 [K]) of the norm whose forward saved h and rstd.

    dy: gradient of the normalised output; dh: gradient that reaches h past the norm (the residual
    stream's), added to dx. dx is the gradient of x and of the residual alike. dy, h, dh and dx have
    one type (bf16 or fp32); dx may be written over any of them. dweight has the same bits in every
    run."""
    if dx is None and dweight is None and _on_gpu(h):
        r = _lib.fast().rms_norm_backward(dy, h, weight, rstd, dh)
        if r is not None:
            return _fast_result(r, "c3cu_rms_norm_bwd")
    code = _dtype_code(h, "h")
    M, K = h.shape
    if K < 1:
        raise _lib.C3CUError(-1, "h", "rows need at least one element")
    dev, dtype = h.get_device(), h.dtype
    ldh = _rows_of(h, "h", dtype, M, K, dev)
    ldy = _rows_of(dy, "dy", dtype, M, K, dev)
    lddh = lddx = K
    if dh is not None:
        lddh = _rows_of(dh, "dh", dtype, M, K, dev)
    _vector_of(weight, "weight", torch.float32, K, dev)
    _vector_of(rstd, "rstd", torch.float32, M, dev)
    if dx is not None:
        lddx = _rows_of(dx, "dx", dtype, M, K, dev)
        _require_same_rows_or_apart(dx, lddx, "dx", ((dy, ldy, "dy"), (h, ldh, "h"), (dh, lddh, "dh")))
        _require_apart(dx, "dx", (weight, "weight"), (rstd, "rstd"))
    else:
        dx = torch.empty(M, K, dtype=dtype, device=h.device)
    if dweight is None:
        dweight = torch.empty(K, dtype=torch.float32, device=h.device)
    else:
        _vector_of(dweight, "dweight", torch.float32, K, dev)
        _require_apart(dweight, "dweight", (dy, "dy"), (h, "h"), (dh, "dh"), (weight, "weight"), (rstd, "rstd"),
                       (dx, "dx"))
    # the workspace is of this call alone: a graph that captures it keeps its own
    if dev == _current_device():
        nb = _lib.load().c3cu_rms_norm_bwd_workspace(M, K)
    else:
        with torch.cuda.device(dev):
            nb = _lib.load().c3cu_rms_norm_bwd_workspace(M, K)
    ws = torch.empty(nb, dtype=torch.uint8, device=h.device) if nb else None
    _call("c3cu_rms_norm_bwd", dev, dy.data_ptr(), ldy, h.data_ptr(), ldh, _ptr(dh), lddh, code, weight.data_ptr(),
          rstd.data_ptr(), dx.data_ptr(), lddx, dweight.data_ptr(), M, K, _ptr(ws), nb)
    return dx, dweight
