"""Rotary positions computed from the positions themselves, for any layout of the pairs.

``prism_b200.producer`` fuses the layer's own form (bf16, whole heads, interleaved pairs, a
stored table) into the all-to-all pack.  ``apply_rotary`` is the operator on its own: bf16,
fp16 or fp32, interleaved or half layout, part of the head, shared key heads, one position
axis or up to three (frame / height / width), positions from a tensor and no table, and its
gradient.  ``rotary_frequencies`` gives the frequencies, scaled for contexts longer than the
trained one.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib

def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, *, scaling: Optional[str] = None,
                       factor: float = 1.0, original_length: Optional[int] = None, beta_fast: float = 32.0,
                       beta_slow: float = 1.0, device=None) -> Tuple[torch.Tensor, float]:
    """(freqs [rotary_dim / 2] fp64, radians per position; the factor on the rotated values).

    scaling None: theta^(-2j / rotary_dim).  For contexts ``factor`` times the trained length:
    * "linear": every frequency divided by factor (positions interpolated);
    * "ntk": the base widened to theta * factor^(rotary_dim / (rotary_dim - 2)), which divides
      the slowest frequency by factor and leaves the fastest;
    * "yarn": pairs that turn more than beta_fast times over original_length keep their
      frequency, those below beta_slow turns are divided by factor, a linear ramp in the pair
      index between; the values are multiplied by 0.1 ln(factor) + 1 (on q and k alike)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even number, got {rotary_dim}")
    if factor < 1.0:
        raise ValueError(f"factor must be at least 1, got {factor}")
    j2 = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs rotary_dim of at least 4")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    freqs = theta ** (-j2 / rotary_dim)
    gain = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "yarn":
        if original_length is None or original_length < 1:
            raise ValueError("yarn scaling needs original_length, the trained context length")
        # pair index at which a frequency turns `beta` times over the original length
        pair = lambda beta: (rotary_dim * math.log(original_length / (beta * 2 * math.pi))) / (2 * math.log(theta))
        # the ramp may end behind the last pair: where that one still turns more than beta_slow times
        low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rotary_dim - 1)
        # high <= 0: even the fastest pair turns no more than beta_slow times
        ramp = ((j2 / 2 - low) / max(high - low, 1e-3)).clamp(0, 1) if high > 0 else torch.ones_like(j2)
        freqs = freqs * (1 - ramp) + freqs / factor * ramp
        gain = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    return freqs.to(device), gain


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor, *,
                 layout: str = "interleaved", sections: Optional[Sequence[int]] = None,
                 scale: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q [S, Hq, D] or [B, S, Hq, D] and k [.., Hk, D] (or None), rotated -> new (q, k).

    The first rot = 2 * len(freqs) columns of each head are rotated by the token's positions,
    the rest copied.  layout "interleaved" pairs columns (2j, 2j + 1), "half" (j, j + rot / 2).
    positions: int32 or int64 [S] or [B, S]; with sections (a, b[, c]), the numbers of pairs
    that follow each axis, [.., S, 2 or 3].  freqs: fp64, radians per position
    (``rotary_frequencies``).  scale multiplies the rotated columns.  Any strides of batch,
    token and head; differentiable in q and k, any number of times."""
    return _lib.torch_ops().apply_rotary(q, k, positions, freqs, layout, sections, scale)


__all__ = ["rotary_frequencies", "apply_rotary"]
