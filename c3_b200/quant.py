"""Activations held in 8 bits: int8 rows with one fp32 scale each, x[m][k] ~ q[m][k] * scale[m].

`quantize_rows` makes that form of an activation (a checkpoint saved for the backward pass) or of
a weight W [N, K] (a scale per output channel); `norm.rms_norm_int8` makes it of a normalised
activation. `linear.forward_int8` multiplies two of them and `linear.grad_weight_int8` takes a
checkpoint back into the weight gradient. The reference has no counterpart (fp32 throughout)."""
from __future__ import annotations

import torch

from . import _lib
from .linear import _call, _fast_result, _on_gpu, _require_apart, _rows_of, _vector_of

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def _dtype_code(t, name: str) -> int:
    if not isinstance(t, torch.Tensor):
        raise _lib.C3CUError(-1, name, f"expected a torch.Tensor, got {type(t).__name__}")
    code = _DTYPES.get(t.dtype)
    if code is None or t.dim() != 2:
        raise _lib.C3CUError(-1, name, f"expected 2-D float32 or bfloat16, got {t.dtype} {tuple(t.shape)}")
    return code


def empty_rows(m: int, k: int, device) -> torch.Tensor:
    """An uninitialised int8 [m, k] whose rows start on 16 bytes, as the int8 GEMMs read them: a column
    slice of a buffer `row_stride(k)` wide, unless k is a multiple of 16."""
    if k % 16 == 0:
        return torch.empty(m, k, dtype=torch.int8, device=device)
    return torch.empty(m, row_stride(k), dtype=torch.int8, device=device)[:, :k]


def row_stride(k: int) -> int:
    return (k + 15) // 16 * 16


def quantize_rows(x: torch.Tensor, q: torch.Tensor | None = None, scale: torch.Tensor | None = None):
    """(q int8 [M, K], scale fp32 [M]) of x [M, K] (bf16 or fp32, unit column stride, any row stride).

    q is the integer nearest to 127 x / A (ties to even) with A the row's largest |x|, scale = A / 127.
    A row of zeros gets scale 0; a row with an infinity or a NaN gets q = 0 and scale NaN."""
    if q is None and scale is None and _on_gpu(x):
        r = _lib.fast().quantize_rows(x)
        if r is not None:
            return _fast_result(r, "c3cu_quantize_rows")
    code = _dtype_code(x, "x")
    M, K = x.shape
    if K < 1:
        raise _lib.C3CUError(-1, "x", "rows need at least one element")
    dev = x.get_device()
    ldx = _rows_of(x, "x", x.dtype, M, K, dev)
    if q is None:
        q, ldq = empty_rows(M, K, x.device), row_stride(K)
    else:
        ldq = _rows_of(q, "q", torch.int8, M, K, dev)
        _require_apart(q, "q", (x, "x"))
    if scale is None:
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
    else:
        _vector_of(scale, "scale", torch.float32, M, dev)
        _require_apart(scale, "scale", (x, "x"), (q, "q"))
    _call("c3cu_quantize_rows", dev, x.data_ptr(), ldx, code, q.data_ptr(), ldq, scale.data_ptr(), M, K)
    return q, scale
