"""Residual addition and RMS norm around the attention and feed-forward layers of a block.

* ``add_rms_norm(x, residual, weight, eps)`` -> (y, h): h = x + residual, rounded to the
  tensors' type, is the residual stream that the next layer adds to, and y its RMS norm times
  weight; one pass, differentiable in x, residual and weight, once: a gradient of y's gradient is an
  error.
* ``add_rms_norm_fp8`` -> (y8, scale, h): the same with y in 8 bits (e4m3) and one fp32 scale a
  row, y ~ y8 * scale, as ``prism_b200.linear.linear_fp8`` reads it.  For inference.
* ``quantize_rows_fp8(x)`` -> (x8, scale): rows (a weight's output features, a layer's input)
  in the same 8-bit form, without a norm.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                 weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """x, residual [..., C] (bf16, fp16 or fp32), weight [C] -> (y, h), both [..., C] in x's type.
    Without a residual h is x."""
    return _lib.torch_ops().add_rms_norm(x, residual, weight, eps)


def add_rms_norm_fp8(x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                     weight: Optional[torch.Tensor] = None,
                     eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """As add_rms_norm, with y as (y8 [..., C] float8_e4m3fn, scale [...] fp32) -> (y8, scale, h).
    scale = max(max |y| / 448, 2^-100) of each row; a row with a NaN or an infinity has scale NaN."""
    return _lib.torch_ops().add_rms_norm_fp8(x, residual, weight, eps, True)


def quantize_rows_fp8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., C] -> (x8 [..., C] float8_e4m3fn, scale [...] fp32), x ~ x8 * scale."""
    return _lib.torch_ops().add_rms_norm_fp8(x, None, None, 0.0, False)[:2]


__all__ = ["add_rms_norm", "add_rms_norm_fp8", "quantize_rows_fp8"]
