"""Activations held in 8 bits: int8 rows with one fp32 scale each, x[m][k] ~ q[m][k] * scale[m].

`quantize_rows` makes that form of an activation (a checkpoint saved for the backward pass) or of
a weight W [N, K] (a scale per output channel); `norm.rms_norm_int8` makes it of a normalised
activation. `linear.forward_int8` multiplies two of them and `linear.grad_weight_int8` takes a
checkpoint back into the weight gradient. The reference has no counterpart (fp32 throughout)."""
from __future__ import annotations

import torch

from . import _lib
from .linear import _ld, _p, _require, _require_rows, _stream

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def _dtype_code(t, name: str) -> int:
    if not isinstance(t, torch.Tensor):
        raise _lib.C3CUError(-1, name, f"expected a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in _DTYPES or t.dim() != 2:
        raise _lib.C3CUError(-1, name, f"expected 2-D float32 or bfloat16, got {t.dtype} {tuple(t.shape)}")
    return _DTYPES[t.dtype]


def empty_rows(m: int, k: int, device) -> torch.Tensor:
    """An uninitialised int8 [m, k] whose rows start on 16 bytes (a column slice of a wider buffer
    unless k is a multiple of 16), as the int8 GEMMs read them."""
    if k % 16 == 0:
        return torch.empty(m, k, dtype=torch.int8, device=device)
    return torch.empty(m, (k + 15) // 16 * 16, dtype=torch.int8, device=device)[:, :k]


@_lib.on_tensor_device
def quantize_rows(x: torch.Tensor, q: torch.Tensor | None = None, scale: torch.Tensor | None = None):
    """(q int8 [M, K], scale fp32 [M]) of x [M, K] (bf16 or fp32, unit column stride, any row stride).

    q is the integer nearest to 127 x / A (ties to even) with A the row's largest |x|, scale = A / 127.
    A row of zeros gets scale 0; a row with an infinity or a NaN gets q = 0 and scale NaN."""
    code = _dtype_code(x, "x")
    M, K = x.shape
    if K < 1:
        raise _lib.C3CUError(-1, "x", "rows need at least one element")
    _require_rows(x, "x", x.dtype, M, K)
    if q is None:
        q = empty_rows(M, K, x.device)
    else:
        _require_rows(q, "q", torch.int8, M, K)
    if scale is None:
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
    else:
        _require(scale, "scale", torch.float32, 1, (M,))
    rc = _lib.load().c3cu_quantize_rows(_p(x), _ld(x), code, _p(q), _ld(q), _p(scale), M, K, _stream(x.device))
    _lib.check(rc, "c3cu_quantize_rows")
    return q, scale
