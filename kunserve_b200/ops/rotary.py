"""Rotary positions: frequencies (plain or scaled for long contexts) and the
rotation, alone or fused with the append to a paged cache.

The kernel takes each pair's frequency in turns per position as a 64-bit
fraction, so the angle of any 32-bit position is exact to the last bits of
its fp32 sine and cosine (``csrc/kernels/rotary.cu``).
"""
import math
from typing import Optional

import torch

from ._native import native

_SCALING_KEYS = {
    "default": set(),
    "linear": {"factor"},
    "dynamic": {"factor", "original_max_position_embeddings"},
    "llama3": {"factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"},
    "yarn": {"factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "attention_factor"},
}
_OPTIONAL = {"beta_fast", "beta_slow", "attention_factor"}


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: Optional[dict] = None,
                       max_position: Optional[int] = None):
    """Radians per position of the ``rotary_dim / 2`` pairs (64-bit CPU
    tensor), and the factor on cos and sin.

    ``scaling`` is the ``rope_scaling`` entry of a HuggingFace config:
    ``linear`` (positions divided by the factor), ``dynamic`` (a larger base
    once ``max_position`` exceeds the original context), ``llama3`` (low
    frequencies divided, high ones kept, a linear mix between) or ``yarn``
    (the same by rotation counts, and a factor on cos and sin).  Other kinds and
    keys (``longrope``, yarn's ``mscale`` and ``truncate``, a ``rope_theta``
    among them) are refused, and so is an original context left to the model's
    other settings: ``original_max_position_embeddings`` must be given where the
    kind needs it."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even number, got {rotary_dim}")
    if not theta > 0:
        raise ValueError(f"theta must be positive, got {theta}")
    pair = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    s = dict(scaling or {})
    kind = s.pop("rope_type", s.pop("type", "default"))
    s.pop("type", None)
    if kind not in _SCALING_KEYS:
        raise ValueError(f"rope scaling {kind!r} is not one of {sorted(_SCALING_KEYS)}")
    unknown, missing = set(s) - _SCALING_KEYS[kind], _SCALING_KEYS[kind] - _OPTIONAL - set(s)
    if unknown or missing:
        raise ValueError(f"rope scaling {kind!r}: unknown keys {sorted(unknown)}, missing keys {sorted(missing)}")
    factor = float(s.get("factor", 1.0))
    if factor < 1.0:
        raise ValueError(f"rope scaling factor must be at least 1, got {factor}")
    old = s.get("original_max_position_embeddings")
    if kind == "dynamic":
        if max_position is None or rotary_dim <= 2:
            raise ValueError("dynamic rope scaling needs max_position and a rotary_dim above 2")
        length = max(max_position, old)
        theta = theta * (factor * length / old - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
    freq = theta ** (-pair / rotary_dim)
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "llama3":
        low, high = float(s["low_freq_factor"]), float(s["high_freq_factor"])
        if high <= low:
            raise ValueError("llama3 rope scaling: high_freq_factor must exceed low_freq_factor")
        turns = old * freq / (2 * math.pi)       # turns of each pair within the original context
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return freq * (keep + (1.0 - keep) / factor), 1.0
    if kind == "yarn":
        if theta <= 1.0:
            raise ValueError("yarn rope scaling needs theta above 1")

        def pair_of(rotations):                  # (fractional) dim that turns so often in the original context
            return rotary_dim * math.log(old / (rotations * 2 * math.pi)) / (2 * math.log(theta))

        low = max(math.floor(pair_of(float(s.get("beta_fast", 32.0)))), 0)
        high = min(math.ceil(pair_of(float(s.get("beta_slow", 1.0)))), rotary_dim - 1)
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        scale = s.get("attention_factor")
        if scale is None:
            scale = 0.1 * math.log(factor) + 1.0
        return freq * (1.0 - ramp) + freq / factor * ramp, float(scale)
    return freq, 1.0


class Rotary:
    """The frequencies of a model's rotary positions, on one device.

    ``rotary_dim`` (default: the whole head) leading dims of each head turn;
    ``interleaved`` pairs dims (2i, 2i + 1) instead of (i, i + rotary_dim / 2)."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, theta: float = 10000.0,
                 interleaved: bool = False, scaling: Optional[dict] = None, max_position: Optional[int] = None,
                 device="cuda"):
        self.head_dim = int(head_dim)
        self.rotary_dim = int(rotary_dim if rotary_dim is not None else head_dim)
        if self.rotary_dim > self.head_dim:
            raise ValueError(f"rotary_dim {self.rotary_dim} exceeds head_dim {self.head_dim}")
        self.interleaved = bool(interleaved)
        self.frequencies, self.scale = rotary_frequencies(self.rotary_dim, theta, scaling, max_position)
        turns = [round(f / (2 * math.pi) * 2 ** 64) % 2 ** 64 for f in self.frequencies.tolist()]
        signed = [t - 2 ** 64 if t >= 2 ** 63 else t for t in turns]
        self.steps = torch.tensor(signed, dtype=torch.int64, device=device)
        self._native = None
        if self.steps.is_cuda:
            self._native = native().RotaryTable(self.steps, self.scale, self.head_dim, self.interleaved)


class _Turn(torch.autograd.Function):
    """The rotation of a tensor whose gradient is asked for: a gradient turns
    back (the map is linear, its transpose the rotation by the opposite angle
    with the same factor)."""

    @staticmethod
    def forward(ctx, x, positions, rotary, inverse):
        ctx.save_for_backward(positions)
        ctx.rotary, ctx.inverse = rotary, inverse
        return native().rotary_apply(x, positions, rotary._native, None, inverse)

    @staticmethod
    def backward(ctx, grad):
        positions, = ctx.saved_tensors
        if grad.stride(-1) != 1:          # broadcast from a sum, say
            grad = grad.contiguous()
        return rotary_apply(grad, positions, ctx.rotary, inverse=not ctx.inverse), None, None, None


def rotary_apply(x: torch.Tensor, positions: torch.Tensor, rotary: Rotary, out: Optional[torch.Tensor] = None,
                 inverse: bool = False) -> torch.Tensor:
    """``x`` [T, heads, head_dim] (bf16 or fp16, any strides between heads and
    tokens) with every head turned to its token's position (int32 [T]).

    ``out`` may be ``x``.  ``inverse`` turns back; with the factor on cos and
    sin kept, that is the gradient: if y = rotary_apply(x), the gradient of x
    is rotary_apply(gradient of y, inverse=True).  Autograd does so where ``x``
    requires a gradient; ``out`` is refused there."""
    y = native().rotary_apply(x, positions, rotary._native, out, inverse)
    return y if y is not None else _Turn.apply(x, positions, rotary, inverse)


def rotary_append(qkv: torch.Tensor, positions: torch.Tensor, pages: torch.Tensor, slots: torch.Tensor,
                  rotary: Rotary, kv, layer: int, out: Optional[torch.Tensor] = None,
                  weights: Optional[torch.Tensor] = None, slot_positions: Optional[torch.Tensor] = None) -> None:
    """Turn the queries and keys of ``qkv`` [T, q heads + 2 kv heads, head_dim]
    and append keys and values to ``layer`` of the cache ``kv`` (``PagedKV``)
    at token t's ``pages[t]``, ``slots[t]`` (int32).

    Turned queries go to ``out`` [T, q heads, head_dim], by default back into
    ``qkv``.  For a cache that evicts by weight, ``weights`` and
    ``slot_positions`` (see ``DecodePlan``) get the new slots' zero weight and
    their token's position.  A page or slot outside the cache is not written;
    ``check_error`` reports it.  Nothing here carries a gradient."""
    native().rotary_append_scaled(qkv, positions, pages, slots, rotary._native, kv, layer, out, weights, slot_positions)
