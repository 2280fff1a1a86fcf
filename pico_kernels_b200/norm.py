"""The RMS norm of a quantized transformer block: the residual's addition, the
norm and the 8-bit input of the next product (``gemm_w8a8``) in one pass over
the row. No counterpart in the reference.
"""

from __future__ import annotations

import torch

from . import _lib
from .gemm_w8a8 import (_FLOATS, as_rows, check_codes_dtype, check_rows, empty_rows, overlaps,
                        row_pitch, written)

__all__ = ["rms_norm_quant"]


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.stride() == b.stride()


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                   residual: torch.Tensor | None = None, dtype: torch.dtype = torch.int8,
                   residual_out: torch.Tensor | None = None):
    """``h = x + residual``; ``y = h / sqrt(mean(h^2) + eps) * weight`` over the
    last dimension; ``y`` quantized per row as ``quantize_rows`` does.

    ``x[..., K]`` fp16, bf16 or fp32; ``residual`` like ``x``; ``weight[K]`` of
    ``x``'s type or fp32. ``h`` is rounded to ``x``'s type (the residual
    stream's), and the norm is that of the rounded value; everything else is
    fp32 up to the codes. Returns ``(codes[..., K], scale[...])``, and with a
    residual ``(codes, scale, h)``, where ``h`` is written to ``residual_out``
    when given (contiguous, like ``x``; ``x`` or ``residual`` itself updates
    the stream in place). A row that holds a NaN or an infinity gets scale NaN
    and codes 0.

    For inference: no gradient passes, ``h`` comes without autograd history even
    where ``x`` or ``residual`` has one. ``residual_out`` counts as modified in place.
    """
    tf = _lib.torch_fast()
    if tf is not None:
        res = tf.rms_norm_quant(x, weight, eps, residual, dtype, residual_out)
        if type(res) is not int:
            return res
        if res > 0:
            _lib.check(res, "rms_norm_quant")
    check_codes_dtype(dtype)
    check_rows(x, "x", _FLOATS)
    _lib.require_cuda(weight)
    K = x.shape[-1]
    if weight.shape != (K,):
        raise _lib.ShapeError(f"weight must be [{K}] (got {tuple(weight.shape)})")
    if weight.dtype not in (x.dtype, torch.float32):
        raise _lib.DtypeError(f"weight must be {x.dtype} or float32 (got {weight.dtype})")
    if residual is None:
        if residual_out is not None:
            raise _lib.ShapeError("residual_out needs a residual")
    else:
        _lib.require_cuda(residual)
        if residual.shape != x.shape:
            raise _lib.ShapeError(f"residual must be {tuple(x.shape)} (got "
                                  f"{tuple(residual.shape)})")
        if residual.dtype != x.dtype:
            raise _lib.DtypeError(f"residual must be {x.dtype} (got {residual.dtype})")
        if residual_out is not None and (
                residual_out.shape != x.shape or residual_out.dtype != x.dtype
                or residual_out.device != x.device or not residual_out.is_contiguous()):
            raise _lib.ShapeError(f"residual_out must be a contiguous {tuple(x.shape)} {x.dtype} "
                                  f"tensor on {x.device}")
        if residual_out is not None and (
                overlaps(residual_out, weight)
                or any(overlaps(residual_out, t) and not _same(residual_out, t)
                       for t in (x, residual))):
            raise _lib.ShapeError("residual_out may be x or residual itself, but not overlap "
                                  "them otherwise")
    _lib.require_same_device(x, weight, residual)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    q = empty_rows(x.shape, dtype, x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    h = None
    if residual is not None:
        h = residual_out if residual_out is not None else torch.empty(
            x.shape, dtype=x.dtype, device=x.device)
    if scale.numel():
        x2, ldx = as_rows(x)
        r2, ldr = as_rows(residual) if residual is not None else (None, 0)
        with _lib.on_device(x):
            _lib.check(_lib.load().pk_rms_norm_quant(
                x2.data_ptr(), _lib.dtype_code(x.dtype), x2.shape[0], K, ldx, _lib.ptr(r2), ldr,
                weight.data_ptr(), _lib.dtype_code(weight.dtype), eps, _lib.ptr(h), K,
                q.data_ptr(), _lib.dtype_code(dtype), row_pitch(K), scale.data_ptr(),
                _lib.stream_of(x)), "rms_norm_quant")
        written(residual_out)
    return (q, scale) if h is None else (q, scale, h)
