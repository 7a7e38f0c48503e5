"""Projections of a decoder layer in 8-bit integers: tokens with one scale
each, weights with one scale per output channel.

    w = ops.Int8Weight.quantize(weight)                       # once, [out, in]
    q, s, h = ops.add_rms_norm_int8(x, norm_weight, eps, residual=h)
    qkv = ops.int8_linear(q, s, w_qkv)
    q, s = ops.quantize_int8(attention)
    x = ops.int8_linear(q, s, w_o)
    q, s = ops.silu_mul_int8(gate, up)                        # views of one projection's output

A row's scale is its largest magnitude / 127 (fp32; the float below where 127
times it would leave the range) and an element's integer the nearest to 127
times it over that magnitude, halves to even; a row of zeros has scale 0.  A
row with a NaN or an infinity, or whose values leave fp32's range on the way,
has scale NaN and integers 0: everything computed of it is NaN.

All run on the current CUDA stream of their tensors' device and allocate what
they return from it.  They serve: results carry no gradient, and arguments that
require one are refused while gradients are recorded, as are arguments with a
forward-mode tangent.
"""
from typing import Optional, Tuple

import torch

from ._native import native


def quantize_int8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rows of ``x`` [T, K] (bf16, fp16 or fp32, any stride between rows)
    as integers int8 [T, K] and scales fp32 [T].  Rows of the integers start on
    16 bytes: where K is no multiple of 16 the tensor is a view of a wider one."""
    return native().quantize_int8(x)


def dequantize_int8(q: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values ``q`` * ``scales`` [T, K] in ``dtype`` (bf16, fp16 or fp32), or
    in ``out`` and its type."""
    return native().dequantize_int8(q, scales, dtype, out)


def add_rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                      residual: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """h = x + residual, and h / sqrt(mean(h^2) + eps) * weight in 8 bits:
    returns (integers, scales, h).

    ``x`` and ``residual`` are bf16 or fp16 [T, K] with any strides between
    rows, ``weight`` [K] is of their type.  h goes to ``out``, which may be
    ``x`` or ``residual``; it is rounded to their type once, the norm is taken of
    the sum before that (the serving engine's own norm is taken of the rounded
    one).  Without a residual h is ``x`` itself."""
    return native().add_rms_norm_int8(x, weight, eps, residual, out)


def silu_mul_int8(gate: torch.Tensor, up: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """silu(gate) * up in 8 bits, (integers, scales), of bf16 or fp16 [T, K]:
    the halves of a merged projection's output are passed as views.  Values are
    within 11 * 2^-24 of themselves, at any gate, before they go to 8 bits."""
    return native().silu_mul_int8(gate, up)


class Int8Weight:
    """A projection's weights [out, in] as ``int8_linear`` reads them: integers
    ``q`` int8 and a scale per output channel, fp32 [out].  Both are copied, the
    integers laid out in blocks; at most 131071 columns, so that 32 bits hold
    every sum."""

    def __init__(self, q: torch.Tensor, scales: torch.Tensor):
        self._native = native().Int8Weight(q, scales)
        self.out_features, self.in_features = self._native.out_features, self._native.in_features
        self.scales, self.device = self._native.scales, self._native.device

    @classmethod
    def quantize(cls, weight: torch.Tensor) -> "Int8Weight":
        """Of weights in bf16, fp16 or fp32, each channel rounded as
        ``quantize_int8`` does."""
        return cls(*quantize_int8(weight.detach()))


def int8_linear(q: torch.Tensor, scales: torch.Tensor, weight: Int8Weight, bias: Optional[torch.Tensor] = None,
                dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(q @ weight^T) * scales * weight's scales + bias, [T, out], of tokens
    ``q`` int8 [T, in] with ``scales`` fp32 [T], in ``dtype`` (bf16, fp16 or
    fp32), or in ``out`` and its type; ``bias`` [out] is of the same type.

    The sums are exact (int32); scales and bias are applied in fp32 and the
    result is rounded once.  Tokens whose rows do not start on 16 bytes are
    copied first (``quantize_int8`` and the others return such that do)."""
    return native().int8_linear(q, scales, weight._native, bias, dtype, out)
