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

from . import ops

LAYOUTS = ("interleaved", "half")


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
        low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rotary_dim // 2 - 1)
        ramp = ((j2 / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        freqs = freqs * (1 - ramp) + freqs / factor * ramp
        gain = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    return freqs.to(device), gain


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, strides, freqs, ends, interleaved, scale):
        ctx.save_for_backward(positions, freqs)
        ctx.meta = (strides, ends, interleaved, scale)
        ctx.set_materialize_grads(False)
        qo, ko = ops.rotary(q, k, positions, strides, freqs, ends, interleaved, scale)
        return qo if k is None else (qo, ko)

    @staticmethod
    def backward(ctx, gq, gk=None):
        positions, freqs = ctx.saved_tensors
        strides, *meta = ctx.meta
        gq, gk = (g if g is None or g.stride(-1) == 1 else g.contiguous() for g in (gq, gk))
        if gq is None and gk is None:
            return (None,) * 8
        # the conjugate rotation, of whichever gradients there are
        a, b = (gk, None) if gq is None else (gq, gk)
        a, b = ops.rotary(a, b, positions, strides, freqs, *meta, conjugate=True)
        dq, dk = (None, a) if gq is None else (a, b)
        return dq, dk, None, None, None, None, None, None


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor, *,
                 layout: str = "interleaved", sections: Optional[Sequence[int]] = None,
                 scale: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q [S, Hq, D] or [B, S, Hq, D] and k [.., Hk, D] (or None), rotated -> new (q, k).

    The first rot = 2 * len(freqs) columns of each head are rotated by the token's positions,
    the rest copied.  layout "interleaved" pairs columns (2j, 2j + 1), "half" (j, j + rot / 2).
    positions: int32 or int64 [S] or [B, S]; with sections (a, b[, c]), the numbers of pairs
    that follow each axis, [.., S, 2 or 3].  freqs: fp64, radians per position
    (``rotary_frequencies``).  scale multiplies the rotated columns.  Any strides of batch,
    token and head; differentiable in q and k."""
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [S, H, D] or [B, S, H, D], got {tuple(q.shape)}")
    *lead, _, D = q.shape
    ops._dtype_code(q, "apply_rotary")
    if k is not None:
        *k_lead, _, k_D = k.shape
        if k_lead != lead or k_D != D or k.dtype != q.dtype:
            raise ValueError("k must have q's batch, tokens, head dim and type")
    if freqs.dtype != torch.float64 or freqs.dim() != 1:
        raise TypeError("freqs must be a float64 vector (rotary_frequencies)")
    pairs = freqs.shape[0]
    if 2 * pairs > D:
        raise ValueError(f"{pairs} pairs do not fit a head of {D} columns")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if sections is None:
        ends, want = (pairs, pairs), lead
    else:
        axes = len(sections)
        if not 1 <= axes <= 3 or min(sections) < 0 or sum(sections) != pairs:
            raise ValueError(f"sections must be 1 to 3 numbers of pairs that add up to {pairs}, got {tuple(sections)}")
        ends = (pairs, pairs) if axes == 1 else (int(sections[0]), int(sections[0]) + int(sections[1]))
        want = lead + [axes]
        if positions.dim() > 0 and axes > 1 and positions.stride(-1) != 1:
            positions = positions.contiguous()
    shape = list(positions.shape)
    if shape != want and shape != want[len(lead) - 1:]:
        raise ValueError(f"positions must have shape {tuple(want)} (the batch may be left out), got {tuple(shape)}")
    # batch and token strides of the positions; one row for every sequence without a batch
    strides = positions.stride()[:len(lead)] if shape == want else positions.stride()[:1]
    strides = strides if len(strides) == 2 else (0, *strides)
    batched = len(lead) == 2
    if q.stride(-1) != 1:
        q = q.contiguous()
    if k is not None and k.stride(-1) != 1:
        k = k.contiguous()
    if not batched:
        q, k = q.unsqueeze(0), None if k is None else k.unsqueeze(0)
    args = (q, k, positions, strides, freqs.contiguous(), ends, layout == "interleaved", float(scale))
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        out = _Rotary.apply(*args)
        qo, ko = (out, None) if k is None else out
    else:
        qo, ko = ops.rotary(*args)
    return (qo, ko) if batched else (qo[0], None if ko is None else ko[0])


__all__ = ["rotary_frequencies", "apply_rotary", "LAYOUTS"]
