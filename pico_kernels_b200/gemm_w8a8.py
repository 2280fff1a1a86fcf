"""W8A8: products of 8-bit activations and 8-bit weights with one scale per
token and one per output channel, on hand-written sm_100a kernels. The
reference has no counterpart (its fp8 product scales whole matrices,
gemm_fp8.py:89-117); the operators follow the manner of ``gemm_int4`` and
``gemm_fp8``.

* ``quantize_rows(x, dtype) -> (codes, scale)``: symmetric quantization of the
  last dimension, one fp32 scale per row (``x ~= codes * scale``), int8 or
  e4m3. Rows of activations are tokens; rows of an ``nn.Linear`` weight
  ``[out, in]`` are output channels, so the same call prepares both operands.
* ``dequantize_rows(codes, scale, dtype)``: the values back.
* ``w8a8_gemm(a8, a_scale, w8, w_scale)``: ``(a8 @ w8^T) * a_scale[m] *
  w_scale[n] (+ bias[n])``; int8 sums are exact (int32).
* ``w8a8_gated_gemm(a8, a_scale, w_gate, gate_scale, w_up, up_scale)``: both
  input projections of a gated feed-forward block, the activation and the
  product in one kernel.

The norm that feeds them is ``norm.rms_norm_quant``; ``linear.W8A8Linear`` and
``linear.W8A8GatedMLP`` run them as modules.

Weights are ``[N, K]`` here (``gemm_int4`` and ``gemm_fp8`` take ``[K, N]``):
the layout ``nn.Linear`` stores and ``quantize_rows`` writes, in which both
operands of an 8-bit product are contiguous along the summed dimension. Codes
are stored with rows a multiple of 16 bytes apart, which the kernels' bulk
loads need; ``quantize_rows`` returns such tensors (a view of its first ``K``
columns when ``K`` is not a multiple of 16), and a product copies operands laid
out otherwise. Everything here is for inference: neither codes nor products have
autograd history, whatever the inputs have; an ``out`` counts as modified in place.
"""

from __future__ import annotations

import torch

from . import _lib

__all__ = ["quantize_rows", "dequantize_rows", "w8a8_gemm", "w8a8_gated_gemm"]

_CODES = (torch.int8, torch.float8_e4m3fn)
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
ACTIVATIONS = {"silu": 0, "gelu_tanh": 1}


def check_codes_dtype(dtype: torch.dtype) -> None:
    if dtype not in _CODES:
        raise _lib.DtypeError(f"8-bit rows are int8 or float8_e4m3fn (got {dtype})")


def check_rows(x: torch.Tensor, what: str, dtypes) -> None:
    _lib.require_cuda(x)
    if x.dtype not in dtypes:
        raise _lib.DtypeError(f"{what} must be one of {', '.join(map(str, dtypes))} "
                              f"(got {x.dtype})")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise _lib.ShapeError(f"{what} needs a last dimension of at least one "
                              f"(got {tuple(x.shape)})")


def as_rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``x`` as 2-D rows with a contiguous last dimension, and the distance
    between them (a view where the strides allow one)."""
    x2 = x.reshape(-1, x.shape[-1])
    if x2.shape[-1] > 1 and x2.stride(1) != 1:
        x2 = x2.contiguous()
    if x2.shape[0] > 1 and x2.stride(0) < x2.shape[1]:  # rows that overlap (an expanded tensor)
        x2 = x2.contiguous()
    return x2, x2.stride(0) if x2.shape[0] > 1 else x2.shape[1]


def empty_rows(shape, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """Storage of 8-bit rows: rows a multiple of 16 bytes apart."""
    K = shape[-1]
    pitch = (K + 15) // 16 * 16
    t = torch.empty((*shape[:-1], pitch), dtype=dtype, device=device)
    return t if pitch == K else t[..., :K]


def row_pitch(K: int) -> int:
    return (K + 15) // 16 * 16


def overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors meet."""
    def span(t: torch.Tensor) -> tuple[int, int]:
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    if a.numel() == 0 or b.numel() == 0 or a.device != b.device:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def written(t: torch.Tensor | None) -> None:
    """Tell autograd that a caller's tensor has new contents: a backward pass that
    saved the old ones then fails (inference tensors are not counted)."""
    if t is not None and not t.is_inference():
        torch.autograd.graph.increment_version(t)


def quantize_rows(x: torch.Tensor, dtype: torch.dtype = torch.int8
                  ) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantize ``x[..., K]`` (fp16, bf16 or fp32) to 8 bits, one scale per row.

    ``scale = max|row|.clamp_min(1e-12) / most`` and ``codes = round(row *
    most / max|row|)``, half steps to even, ``most`` = 127 for int8 and 448 for
    ``float8_e4m3fn``. Codes of 16-bit rows are the nearest there are; of fp32
    rows a quotient within 2^-24 of its size from a midpoint may take either
    side. Returns ``(codes[..., K], scale[...] fp32)`` with ``x ~= codes *
    scale``. A row that holds a NaN or an infinity gets scale NaN and codes 0:
    its products are NaN, other rows' are not.
    """
    tf = _lib.torch_fast()
    if tf is not None:
        res = tf.quantize_rows(x, dtype)
        if type(res) is not int:
            return res
        if res > 0:
            _lib.check(res, "quantize_rows")
    check_codes_dtype(dtype)
    check_rows(x, "x", _FLOATS)
    K = x.shape[-1]
    q = empty_rows(x.shape, dtype, x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if scale.numel() == 0:
        return q, scale
    x2, ldx = as_rows(x)
    with _lib.on_device(x):
        _lib.check(_lib.load().pk_quantize_rows(
            x2.data_ptr(), _lib.dtype_code(x.dtype), x2.shape[0], K, ldx, q.data_ptr(),
            _lib.dtype_code(dtype), row_pitch(K), scale.data_ptr(), _lib.stream_of(x)),
            "quantize_rows")
    return q, scale


def dequantize_rows(q: torch.Tensor, scale: torch.Tensor,
                    dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``q[..., K] * scale[..., None]`` in fp32, rounded once to ``dtype``
    (fp32, bf16 or fp16)."""
    tf = _lib.torch_fast()
    if tf is not None:
        res = tf.dequantize_rows(q, scale, dtype)
        if type(res) is not int:
            return res
        if res > 0:
            _lib.check(res, "dequantize_rows")
    check_rows(q, "codes", _CODES)
    if dtype not in _FLOATS:
        raise _lib.DtypeError(f"dequantize_rows writes fp16, bf16 or fp32 (got {dtype})")
    scale = _scale(scale, q.shape[:-1], q, "scale")
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    if out.numel() == 0:
        return out
    q2, ldq = as_rows(q)
    K = q.shape[-1]
    with _lib.on_device(q):
        _lib.check(_lib.load().pk_dequantize_rows(
            q2.data_ptr(), _lib.dtype_code(q.dtype), q2.shape[0], K, ldq, scale.data_ptr(),
            out.data_ptr(), _lib.dtype_code(dtype), K, _lib.stream_of(q)), "dequantize_rows")
    return out


def _scale(s: torch.Tensor, shape, like: torch.Tensor, what: str) -> torch.Tensor:
    """A contiguous fp32 tensor of one value per row (a trailing 1 is allowed)."""
    _lib.require_cuda(s)
    _lib.require_same_device(like, s)
    if s.dtype != torch.float32:
        raise _lib.DtypeError(f"{what} must be float32 (got {s.dtype})")
    if tuple(s.shape) not in (tuple(shape), (*shape, 1)):
        raise _lib.ShapeError(f"{what} must be {tuple(shape)}: one value per row "
                              f"(got {tuple(s.shape)})")
    return s if s.is_contiguous() else s.contiguous()


def _codes(t: torch.Tensor, dtype: torch.dtype | None, what: str) -> tuple[torch.Tensor, int]:
    """A 2-D operand the kernels can load (16-byte aligned rows), and its pitch."""
    check_rows(t, what, _CODES)
    if dtype is not None and t.dtype != dtype:
        raise _lib.DtypeError(f"operands must be both int8 or both e4m3 ({what} is {t.dtype})")
    if t.dim() != 2:
        raise _lib.ShapeError(f"{what} must be 2-D (got {tuple(t.shape)})")
    rows, K = t.shape
    pitch = t.stride(0) if rows > 1 else row_pitch(K)
    if ((K > 1 and t.stride(1) != 1) or pitch % 16 or pitch < K or t.data_ptr() % 16):
        c = empty_rows((rows, K), t.dtype, t.device)
        c.copy_(t)
        return c, row_pitch(K)
    return t, pitch


def _out(M: int, N: int, out_dtype: torch.dtype, out: torch.Tensor | None,
         device: torch.device, operands) -> torch.Tensor:
    if out_dtype not in _FLOATS:
        raise _lib.DtypeError(f"output must be fp32, bf16 or fp16 (got {out_dtype})")
    if out is None:
        return torch.empty((M, N), dtype=out_dtype, device=device)
    if (out.shape != (M, N) or out.dtype != out_dtype or out.device != device
            or not out.is_contiguous()):
        raise _lib.ShapeError(f"out must be a contiguous [{M}, {N}] {out_dtype} tensor on "
                              f"{device}")
    if any(t is not None and overlaps(out, t) for t in operands):
        raise _lib.ShapeError("out must not overlap an operand: they are read while it is written")
    return out


def w8a8_gemm(a8: torch.Tensor, a_scale: torch.Tensor, w8: torch.Tensor, w_scale: torch.Tensor, *,
              bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """``(a8[M, K] @ w8[N, K]^T) * a_scale[m] * w_scale[n] (+ bias[n])``.

    ``a8`` and ``w8``: both int8 (summed exactly in int32; K <= 131071) or both
    ``float8_e4m3fn`` (fp32 sums; K <= 2^24), as ``quantize_rows`` returns them;
    ``a_scale[M]``, ``w_scale[N]`` and ``bias[N]`` fp32. The scales and the
    bias are applied in fp32 in the epilogue and the result rounded once to
    ``out_dtype`` (fp32, bf16 or fp16), into ``out`` when given (a contiguous
    ``[M, N]`` tensor of ``out_dtype`` that overlaps no operand). No workspace and no host
    synchronisation: calls can be captured in CUDA graphs.
    """
    tf = _lib.torch_fast()
    if tf is not None:
        res = tf.w8a8_gemm(a8, a_scale, w8, w_scale, bias, out_dtype, out)
        if type(res) is not int:
            return res
        if res > 0:
            _lib.check(res, "w8a8_gemm")
    a, lda = _codes(a8, None, "a8")
    w, ldw = _codes(w8, a.dtype, "w8")
    _lib.require_same_device(a, w)
    M, K = a.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise _lib.ShapeError(f"inner dimensions differ: a8 has K={K}, w8 has K={w.shape[1]}")
    sa = _scale(a_scale, (M,), a, "a_scale")
    sw = _scale(w_scale, (N,), a, "w_scale")
    b = None if bias is None else _scale(bias, (N,), a, "bias")
    y = _out(M, N, out_dtype, out, a.device, (a, sa, w, sw, b))
    if y.numel() == 0:
        return y
    with _lib.on_device(a):
        _lib.check(_lib.load().pk_w8a8_gemm(
            a.data_ptr(), _lib.dtype_code(a.dtype), lda, sa.data_ptr(), w.data_ptr(), ldw,
            sw.data_ptr(), _lib.ptr(b), M, N, K, y.data_ptr(), _lib.dtype_code(out_dtype), N,
            _lib.stream_of(a)), "w8a8_gemm")
    written(out)
    return y


def w8a8_gated_gemm(a8: torch.Tensor, a_scale: torch.Tensor, w_gate: torch.Tensor,
                    gate_scale: torch.Tensor, w_up: torch.Tensor, up_scale: torch.Tensor, *,
                    activation: str = "silu", out_dtype: torch.dtype = torch.float32,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """``act(g) * u`` with ``g`` and ``u`` the products ``w8a8_gemm`` defines
    for ``w_gate[N, K]`` and ``w_up[N, K]``, in one kernel that writes only the
    ``[M, N]`` result.

    ``activation``: ``"silu"`` (``g * sigmoid(g)``) or ``"gelu_tanh"`` (GELU's
    tanh form). ``g``, ``u`` and the activation are fp32, rounded once to
    ``out_dtype``; the other arguments are ``w8a8_gemm``'s.
    """
    tf = _lib.torch_fast()
    if tf is not None:
        res = tf.w8a8_gated_gemm(a8, a_scale, w_gate, gate_scale, w_up, up_scale,
                                 ACTIVATIONS.get(activation, -1), out_dtype, out)
        if type(res) is not int:
            return res
        if res > 0:
            _lib.check(res, "w8a8_gated_gemm")
    if activation not in ACTIVATIONS:
        raise _lib.ShapeError(f"activation must be one of {', '.join(ACTIVATIONS)} "
                              f"(got {activation!r})")
    a, lda = _codes(a8, None, "a8")
    g, ldg = _codes(w_gate, a.dtype, "w_gate")
    u, ldu = _codes(w_up, a.dtype, "w_up")
    _lib.require_same_device(a, g, u)
    M, K = a.shape
    N = g.shape[0]
    if g.shape[1] != K or u.shape[1] != K:
        raise _lib.ShapeError(f"inner dimensions differ: a8 has K={K}, w_gate "
                              f"K={g.shape[1]}, w_up K={u.shape[1]}")
    if u.shape[0] != N:
        raise _lib.ShapeError(f"w_gate has {N} channels, w_up {u.shape[0]}")
    sa = _scale(a_scale, (M,), a, "a_scale")
    sg = _scale(gate_scale, (N,), a, "gate_scale")
    su = _scale(up_scale, (N,), a, "up_scale")
    y = _out(M, N, out_dtype, out, a.device, (a, sa, g, sg, u, su))
    if y.numel() == 0:
        return y
    with _lib.on_device(a):
        _lib.check(_lib.load().pk_w8a8_gated_gemm(
            a.data_ptr(), _lib.dtype_code(a.dtype), lda, sa.data_ptr(), g.data_ptr(), ldg,
            sg.data_ptr(), u.data_ptr(), ldu, su.data_ptr(), ACTIVATIONS[activation], M, N, K,
            y.data_ptr(), _lib.dtype_code(out_dtype), N, _lib.stream_of(a)), "w8a8_gated_gemm")
    written(out)
    return y
