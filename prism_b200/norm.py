"""Residual addition and RMS norm around the attention and feed-forward layers of a block.

* ``add_rms_norm(x, residual, weight, eps)`` -> (y, h): h = x + residual, rounded to the
  tensors' type, is the residual stream that the next layer adds to, and y its RMS norm times
  weight; one pass, differentiable in x, residual and weight.
* ``add_rms_norm_fp8`` -> (y8, scale, h): the same with y in 8 bits (e4m3) and one fp32 scale a
  row, y ~ y8 * scale, as ``prism_b200.linear.linear_fp8`` reads it.  For inference.
* ``quantize_rows_fp8(x)`` -> (x8, scale): rows (a weight's output features, a layer's input)
  in the same 8-bit form, without a norm.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, rstd = ops.add_rms_norm(x, residual, weight, eps, want_rstd=True)
        ctx.save_for_backward(x if residual is None else h, rstd, weight)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, gy, gh=None):
        h, rstd, weight = ctx.saved_tensors
        want_x, want_r, want_w = ctx.needs_input_grad[:3]
        if gy is None:  # y is unused: h = x + residual passes its gradient through
            dx, dw = gh, None
        else:
            dx, dw = ops.add_rms_norm_bwd(gy, h, rstd, gh, weight, want_dweight=want_w)
        return (dx if want_x else None, dx if want_r else None,
                dw.to(weight.dtype) if dw is not None else None, None)


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                 weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """x, residual [..., C] (bf16, fp16 or fp32), weight [C] -> (y, h), both [..., C] in x's type.
    Without a residual h is x."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        out = _AddRmsNorm.apply(x, residual, weight, float(eps))
    else:
        y, h, _ = ops.add_rms_norm(x, residual, weight, eps)
        out = y if residual is None else (y, h)
    return (out, x) if residual is None else out


def _no_grad_only(what, *ts):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise NotImplementedError(f"{what} is inference only: its 8-bit rounding has no gradient")


def add_rms_norm_fp8(x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                     weight: Optional[torch.Tensor] = None,
                     eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """As add_rms_norm, with y as (y8 [..., C] float8_e4m3fn, scale [...] fp32) -> (y8, scale, h).
    scale = max(max |y| / 448, 2^-100) of each row; a row with a NaN or an infinity has scale NaN."""
    _no_grad_only("add_rms_norm_fp8", x, residual, weight)
    y8, scale, h = ops.add_rms_norm_fp8(x, residual, weight, eps)
    return y8, scale, x if h is None else h


def quantize_rows_fp8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., C] -> (x8 [..., C] float8_e4m3fn, scale [...] fp32), x ~ x8 * scale."""
    _no_grad_only("quantize_rows_fp8", x)
    x8, scale, _ = ops.add_rms_norm_fp8(x, normalize=False)
    return x8, scale


__all__ = ["add_rms_norm", "add_rms_norm_fp8", "quantize_rows_fp8"]
