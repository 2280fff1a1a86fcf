"""Quantized ``nn.Linear`` drop-ins: W4A16 over the packed-int4 GEMM, and W8A8
over the 8-bit products (``W8A8Linear``, ``W8A8GatedMLP``, below).

The reference quantizes the transformer's ``nn.Linear`` layers in place
(quantize.py:124-129 selects them, quantize.py:160-184 swaps in fake-quant
weights) and then runs them as dense float layers. ``W4A16Linear`` instead
keeps each layer's weight as packed int4 codes plus group scales and runs
``int4_gemm`` on every call, so the weights stream from HBM at 4 bits:

* ``weight[out, in]`` is stored transposed, as the GEMM's ``B[K = in, N = out]``:
  ``w_packed`` uint8 ``[in, out // 2]`` (``pack_int4_n`` layout) and ``scales``
  ``[ceil(in / group_size), out]`` in the activation dtype; symmetric
  round-to-nearest per group of ``group_size`` input features
  (``quantize_int4_grouped``: ``scale = max|w| / 7``, codes in [-7, 7]).
* ``forward(x)`` flattens the leading dimensions of ``x[..., in]`` into M rows
  and computes ``x @ W^T + bias`` with fp32 accumulation; the result has
  ``x``'s dtype, like ``nn.Linear``. M = 1 runs the CUDA-core GEMV, small M the
  tensor-core decode, large M the tcgen05 prefill path.

``W8A8Linear`` holds the weight as 8-bit codes ``[out, in]`` (int8 or e4m3) with
one scale per output channel and quantizes its input per token on every call;
``W8A8GatedMLP`` runs a gated feed-forward block on such weights: norm with the
residual's addition, both input projections with the activation and product in
one kernel, and the output projection. Quantized weights take no gradient, and
W8A8 layers pass none on to their inputs.

``quantize_linear_layers(model)`` swaps every (or every selected) ``nn.Linear``
of a module tree for a ``W4A16Linear`` (or, with ``scheme="w8a8"``, a
``W8A8Linear``) in place.
"""

from __future__ import annotations

from typing import Callable

import torch
import torch.nn as nn

from . import _lib
from .gemm_int4 import int4_gemm, quantize_int4_grouped
from .gemm_w8a8 import (ACTIVATIONS, check_codes_dtype, dequantize_rows, quantize_rows, row_pitch,
                        w8a8_gated_gemm, w8a8_gemm)
from .norm import rms_norm_quant

__all__ = ["W4A16Linear", "W8A8Linear", "W8A8GatedMLP", "quantize_linear_layers"]


class W4A16Linear(nn.Module):
    """``y = x @ W^T + b`` with W held as packed int4 codes and group scales."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 group_size: int = 128, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str | None = None) -> None:
        super().__init__()
        if out_features % 2:
            raise _lib.ShapeError(f"out_features must be even to pack two codes per byte "
                                  f"(got {out_features})")
        if dtype not in (torch.float16, torch.bfloat16):
            raise _lib.DtypeError(f"activation dtype must be fp16 or bf16 (got {dtype})")
        self.in_features = in_features
        self.out_features = out_features
        self.group_size = group_size
        self.dtype = dtype
        groups = (in_features + group_size - 1) // group_size
        self.register_buffer("w_packed", torch.zeros((in_features, out_features // 2),
                                                     dtype=torch.uint8, device=device))
        self.register_buffer("scales", torch.zeros((groups, out_features), dtype=dtype,
                                                   device=device))
        if bias:
            self.register_buffer("bias", torch.zeros(out_features, dtype=torch.float32,
                                                     device=device))
        else:
            self.bias = None
        # act_order GPTQ: the packed rows follow this order of the input features
        self.register_buffer("perm", None)

    @classmethod
    def from_linear(cls, linear: nn.Linear, group_size: int = 128,
                    dtype: torch.dtype | None = None, calib: torch.Tensor | None = None,
                    damp: float = 0.01, act_order: bool = False) -> "W4A16Linear":
        """Quantize ``linear.weight`` (on a CUDA device) into a new layer.

        Round-to-nearest per group by default; with calibration inputs
        ``calib[..., in]`` (this layer's inputs) the GPTQ producer
        (``gptq.gptq_quantize_int4``) chooses the codes. ``dtype``
        (activations and stored scales) defaults to the weight's dtype when
        that is fp16/bf16, else bf16. The bias is kept in fp32. With
        ``act_order`` (GPTQ only) the input features are quantized in order of
        decreasing activation energy (quantize.py:97-101) and stored in that
        order; ``forward`` gathers its inputs with the same permutation.
        """
        w = linear.weight.detach()
        _lib.require_cuda(w)
        if dtype is None:
            dtype = w.dtype if w.dtype in (torch.float16, torch.bfloat16) else torch.bfloat16
        layer = cls(linear.in_features, linear.out_features, linear.bias is not None,
                    group_size, dtype, w.device)
        # group absmax from the weights as stored (fp32 kept exact), scales rounded
        # to the activation dtype as the GEMM reads them
        if calib is not None:
            from .gptq import gptq_quantize_int4
            res = gptq_quantize_int4(w, calib, group_size=group_size, damp=damp,
                                     scale_dtype=dtype, act_order=act_order)
            packed, scales = res[0], res[1]
            if act_order:
                layer.perm = res[2]
        elif act_order:
            raise _lib.ShapeError("act_order needs calibration inputs (GPTQ)")
        else:
            packed, scales = quantize_int4_grouped(w.t(), group_size, scale_dtype=dtype)
        layer.w_packed.copy_(packed)
        layer.scales.copy_(scales)
        if linear.bias is not None:
            layer.bias.copy_(linear.bias.detach().float())
        return layer

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise _lib.ShapeError(f"expected {self.in_features} input features, got {x.shape[-1]}")
        lead = x.shape[:-1]
        x2 = x.reshape(-1, self.in_features)
        if x2.dtype != self.dtype:
            x2 = x2.to(self.dtype)
        if self.perm is not None:
            x2 = x2.index_select(1, self.perm)
        out_dtype = x.dtype if (self.bias is None and x.dtype == torch.bfloat16) else torch.float32
        y = int4_gemm(x2, self.w_packed, self.scales, group_size=self.group_size,
                      out_dtype=out_dtype)
        if self.bias is not None:
            y = y + self.bias
        return y.to(x.dtype).reshape(*lead, self.out_features)

    def dequantized_weight(self) -> torch.Tensor:
        """fp32 ``W[out, in]`` the layer computes with (codes x group scales)."""
        from .gemm_int4 import unpack_int4_n
        q = unpack_int4_n(self.w_packed).float()
        s = self.scales.float().repeat_interleave(self.group_size, dim=0)[: self.in_features]
        w = (q * s).t()
        if self.perm is not None:
            w = w[:, torch.argsort(self.perm)]
        return w.contiguous()

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, group_size={self.group_size}, int4")


class W8A8Linear(nn.Module):
    """``y = x @ W^T + b`` with W in 8-bit codes, one scale per output channel,
    and x quantized to the same 8-bit type per row (token) on every call.

    For inference: the output has no autograd history even where ``x`` has one, so
    nothing before the layer gets a gradient through it."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 dtype: torch.dtype = torch.int8,
                 device: torch.device | str | None = None) -> None:
        super().__init__()
        check_codes_dtype(dtype)
        self.in_features = in_features
        self.out_features = out_features
        self.dtype = dtype
        # rows padded to the pitch the kernels load: a view of them stays as laid
        # out when the module moves between devices
        self.register_buffer("codes", torch.zeros((out_features, row_pitch(in_features)),
                                                  dtype=dtype, device=device))
        self.register_buffer("scales", torch.zeros(out_features, dtype=torch.float32,
                                                   device=device))
        if bias:
            self.register_buffer("bias", torch.zeros(out_features, dtype=torch.float32,
                                                     device=device))
        else:
            self.bias = None

    @classmethod
    def from_linear(cls, linear: nn.Linear, dtype: torch.dtype = torch.int8) -> "W8A8Linear":
        """Quantize ``linear.weight`` (on a CUDA device) per output channel, to
        int8 or ``torch.float8_e4m3fn``. The bias is kept in fp32."""
        w = linear.weight.detach()
        _lib.require_cuda(w)
        layer = cls(linear.in_features, linear.out_features, linear.bias is not None, dtype,
                    w.device)
        codes, scales = quantize_rows(w, dtype)
        layer.weight8.copy_(codes)
        layer.scales.copy_(scales)
        if linear.bias is not None:
            layer.bias.copy_(linear.bias.detach().float())
        return layer

    def _apply(self, fn, recurse: bool = True):
        # Module.to(dtype), half() and the like move the layer and leave its types:
        # a cast would lose the scales and, e4m3 being a floating type, the codes.
        before = dict(self._buffers)
        super()._apply(fn, recurse)
        for name, old in before.items():
            new = self._buffers[name]
            if old is not None and new.dtype != old.dtype:
                self._buffers[name] = old.to(new.device)
        return self

    @property
    def weight8(self) -> torch.Tensor:
        """The codes ``[out, in]`` (a view of their padded storage)."""
        return self.codes[:, : self.in_features]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise _lib.ShapeError(f"expected {self.in_features} input features, got {x.shape[-1]}")
        codes, scale = quantize_rows(x.reshape(-1, self.in_features), self.dtype)
        return self.product(codes, scale, x.dtype).reshape(*x.shape[:-1], self.out_features)

    def product(self, codes: torch.Tensor, scale: torch.Tensor,
                out_dtype: torch.dtype) -> torch.Tensor:
        """The layer on inputs that are quantized already (``quantize_rows``,
        ``rms_norm_quant``): ``codes[M, in]`` and ``scale[M]`` to ``[M, out]``."""
        return w8a8_gemm(codes, scale, self.weight8, self.scales, bias=self.bias,
                         out_dtype=out_dtype)

    def dequantized_weight(self) -> torch.Tensor:
        """fp32 ``W[out, in]`` the layer computes with (codes x channel scales)."""
        return dequantize_rows(self.weight8, self.scales)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, {str(self.dtype).removeprefix('torch.')}")


class W8A8GatedMLP(nn.Module):
    """Gated feed-forward block on 8-bit weights:
    ``down(act(gate(n)) * up(n))`` with ``n`` the block's input, or its RMS norm
    when the block holds a norm weight.

    Four launches a call: the norm (or the quantizer) that writes 8-bit rows, the
    gated product, the quantizer of its result, and the output product. For
    inference: neither the output nor ``h`` has autograd history.
    """

    def __init__(self, gate: W8A8Linear, up: W8A8Linear, down: W8A8Linear,
                 norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 activation: str = "silu") -> None:
        super().__init__()
        if activation not in ACTIVATIONS:
            raise _lib.ShapeError(f"activation must be one of {', '.join(ACTIVATIONS)} "
                                  f"(got {activation!r})")
        if gate.bias is not None or up.bias is not None:
            raise _lib.ShapeError("the gated product has no bias in its input projections")
        if gate.in_features != up.in_features or gate.out_features != up.out_features:
            raise _lib.ShapeError("gate and up must have the same sizes")
        if down.in_features != gate.out_features:
            raise _lib.ShapeError(f"down takes {down.in_features} features, the gated product "
                                  f"gives {gate.out_features}")
        if gate.dtype != up.dtype:
            raise _lib.DtypeError("gate and up must have the same 8-bit type")
        if norm_weight is not None and norm_weight.shape != (gate.in_features,):
            raise _lib.ShapeError(f"norm_weight must be [{gate.in_features}] "
                                  f"(got {tuple(norm_weight.shape)})")
        self.gate, self.up, self.down = gate, up, down
        self.eps = eps
        self.activation = activation
        self.register_buffer("norm_weight", norm_weight)

    @classmethod
    def from_linears(cls, gate: nn.Linear, up: nn.Linear, down: nn.Linear,
                     norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                     activation: str = "silu",
                     dtype: torch.dtype = torch.int8) -> "W8A8GatedMLP":
        """Quantize the three projections (``W8A8Linear.from_linear``)."""
        return cls(*(W8A8Linear.from_linear(m, dtype) for m in (gate, up, down)),
                   norm_weight=None if norm_weight is None else norm_weight.detach(), eps=eps,
                   activation=activation)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        """``x[..., in]`` to ``[..., out]`` in ``x``'s type. With ``residual``
        (blocks with a norm only) the norm is that of ``h = x + residual`` and
        ``(output, h)`` is returned, ``h`` being the residual stream after it."""
        if x.shape[-1] != self.gate.in_features:
            raise _lib.ShapeError(f"expected {self.gate.in_features} input features, got "
                                  f"{x.shape[-1]}")
        if residual is not None and self.norm_weight is None:
            raise _lib.ShapeError("a residual needs a block with a norm")
        x2 = x.reshape(-1, x.shape[-1])
        h = None
        if self.norm_weight is None:
            q, s = quantize_rows(x2, self.gate.dtype)
        elif residual is None:
            q, s = rms_norm_quant(x2, self.norm_weight, self.eps, dtype=self.gate.dtype)
        else:
            if residual.shape != x.shape:
                raise _lib.ShapeError(f"residual must be {tuple(x.shape)} (got "
                                      f"{tuple(residual.shape)})")
            q, s, h = rms_norm_quant(x2, self.norm_weight, self.eps,
                                     residual=residual.reshape(x2.shape), dtype=self.gate.dtype)
        # the block's own type for the hidden values, which the quantizer reads next
        y = w8a8_gated_gemm(q, s, self.gate.weight8, self.gate.scales, self.up.weight8,
                            self.up.scales, activation=self.activation, out_dtype=x.dtype)
        q, s = quantize_rows(y, self.down.dtype)
        out = self.down.product(q, s, x.dtype).reshape(*x.shape[:-1], self.down.out_features)
        return out if h is None else (out, h.reshape(x.shape))

    def extra_repr(self) -> str:
        return f"activation={self.activation}, norm={self.norm_weight is not None}"


def _capture_inputs(model: nn.Module, module: nn.Module, calib) -> torch.Tensor:
    """Inputs ``module`` sees when ``model`` runs on ``calib`` (a tensor or a
    tuple of positional arguments), flattened to ``[rows, in]``
    (quantize.py:132-157)."""
    seen: list[torch.Tensor] = []

    def hook(_m, args):
        seen.append(args[0].detach())

    handle = module.register_forward_pre_hook(hook)
    try:
        with torch.no_grad():
            model(*calib) if isinstance(calib, tuple) else model(calib)
    finally:
        handle.remove()
    return torch.cat([t.reshape(-1, t.shape[-1]) for t in seen], dim=0)


def quantize_linear_layers(model: nn.Module, group_size: int = 128,
                           select: Callable[[str, nn.Linear], bool] | None = None,
                           dtype: torch.dtype | None = None, calib=None,
                           damp: float = 0.01, act_order: bool = False, *,
                           scheme: str = "w4a16") -> nn.Module:
    """Replace ``nn.Linear`` children in place with ``W4A16Linear``, or with
    ``scheme="w8a8"`` by ``W8A8Linear`` (``dtype`` then is the 8-bit type, int8 by
    default; no groups, no calibration; any ``out_features``).

    ``select(name, module)`` picks the layers (default: every ``nn.Linear``
    with an even ``out_features``); quantize.py:124-129 picks those under
    ``transformer.h``, which ``select=lambda n, m: n.startswith("transformer.h")``
    reproduces. With ``calib`` (the model's input: a tensor or a tuple of
    arguments) each layer is GPTQ-quantized from the inputs it sees when the
    model, with the layers before it already quantized, runs on ``calib``
    (the sequential re-capture of quantize.py:160-184); without it, per-group
    round-to-nearest. Returns ``model``.
    """
    if scheme not in ("w4a16", "w8a8"):
        raise _lib.ShapeError(f"scheme must be w4a16 or w8a8 (got {scheme!r})")
    w8a8 = scheme == "w8a8"
    if w8a8:
        if calib is not None or act_order:
            raise _lib.ShapeError("w8a8 rounds to nearest: no calibration, no act_order")
        check_codes_dtype(torch.int8 if dtype is None else dtype)
    targets = [name for name, mod in model.named_modules()
               if isinstance(mod, nn.Linear) and (w8a8 or mod.out_features % 2 == 0)
               and (select is None or select(name, mod))]
    for name in targets:
        parent = model
        *path, leaf = name.split(".")
        for p in path:
            parent = getattr(parent, p)
        mod = getattr(parent, leaf)
        if w8a8:
            setattr(parent, leaf, W8A8Linear.from_linear(mod, torch.int8 if dtype is None else dtype))
            continue
        x = _capture_inputs(model, mod, calib) if calib is not None else None
        setattr(parent, leaf, W4A16Linear.from_linear(mod, group_size, dtype, calib=x, damp=damp,
                                                      act_order=act_order and x is not None))
    return model
