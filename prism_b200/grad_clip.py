"""Global gradient norm over many tensors, and clipping, without a host synchronisation."""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import _lib, ops

def _flat_order(g: torch.Tensor, o: torch.Tensor):
    """(g, o) with their dimensions permuted so that both are contiguous, or None: elements of
    dense tensors with the same shape and strides match one to one in memory order."""
    if g.is_contiguous() and o.is_contiguous():
        return g, o
    if g.shape != o.shape:
        return None
    order = sorted(range(g.dim()), key=lambda d: (-g.stride(d), d))
    gp, op = g.permute(order), o.permute(order)
    return (gp, op) if gp.is_contiguous() and op.is_contiguous() else None


def _check(grads, outs) -> None:
    """What the kernel asks of each tensor, with the error that says so."""
    ops._check_cuda(*grads, *outs)
    for g, o in zip(grads, outs):
        if g.device != grads[0].device or o.device != g.device:
            raise ValueError("gradients and outputs must be on one device")
        if g.dtype not in (torch.bfloat16, torch.float16, torch.float32):
            raise TypeError(f"clip_grad_norm expects bf16, fp16 or fp32, got {g.dtype}")
        if o.dtype != g.dtype or o.numel() != g.numel():
            raise ValueError("an output must have the type and the number of elements of its gradient")


def clip_grad_norm(grads: Sequence[torch.Tensor], max_norm: float, *,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """norm = sqrt(sum of the squares of every element of every gradient) -> 0-dim fp32 tensor on
    the gradients' device; the gradients become g * min(1, max_norm / (norm + 1e-6)), in place or
    in ``out``: for each gradient a tensor of its type and number of elements (its own shape, or
    its slice of a flat buffer, filled in row-major order) that overlaps none of them and no other
    output.  A gradient that is given again in place (one tensor as the gradient of two inputs)
    counts each time and is scaled once; other overlaps of what is written are refused.  bf16,
    fp16 and fp32 gradients may be mixed.  A norm that is not a number makes every gradient NaN;
    max_norm = inf only measures the norm."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be a number that is not negative, got {max_norm}")
    outs = grads
    if out is not None:
        outs = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(outs) != len(grads):
            raise ValueError(f"{len(grads)} gradients, {len(outs)} outputs")
    if not grads:
        return torch.zeros(())
    norm = _lib.torch_ops().clip_grad_norm(grads, outs, max_norm)
    if norm is not None:
        return norm
    _check(grads, outs)
    src, dst, copies = [], [], []
    with torch.no_grad():
        for g, o in zip(grads, outs):
            pair = _flat_order(g, o)
            if pair is None:  # gaps in memory, or two orders: through a contiguous copy
                pair = (g.clone(memory_format=torch.contiguous_format),) * 2
                if out is not None or max_norm != math.inf:
                    copies.append((o, pair[1]))
            src.append(pair[0])
            dst.append(pair[1])
        norm = _lib.torch_ops().clip_grad_norm(src, dst, max_norm)
        for o, c in copies:
            o.copy_(c.view(o.shape))
    return norm


__all__ = ["clip_grad_norm"]
