"""Dense attention over sequences of different lengths that lie one after the other, without padding:
prompts (causal, with grouped heads), their next parts behind keys that are there already, and the
cross-attention of one set of sequences to another.

The block-sparse paths (``prism_b200.dynamic_block_attention``, ``prism_b200.bsa_interface``) attend the
chosen tiles of one long video sequence; ``packed_attention`` attends every key that the mask leaves.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
                     k_offsets: Optional[torch.Tensor] = None, *, causal: bool = True,
                     scale: Optional[float] = None) -> torch.Tensor:
    """q [T, Hq, D], k and v [Tk, Hk, D] -> [T, Hq, D]: softmax(scale q k^T) v within each sequence.

    D is 64 or 128; bf16, or fp16 without gradients.  Query heads h * Hq / Hk .. share key head h (Hq a
    multiple of Hk, up to 128 heads a key head).  Sequence b is the rows offsets[b] .. offsets[b + 1] - 1 of q
    and, by k_offsets (default: offsets), of k and v: int32 or int64 [sequences + 1] on the device, never read
    by the host; non-decreasing, from 0 to the number of rows at most, else the result is NaN.  A sequence may
    be empty on either side.

    causal: with n queries and m keys, query i attends keys 0 .. i + m - n, so the last query attends all of
    them (a prompt has m = n; its next part n < m).  A query without a key gives 0, and so do rows behind the
    last sequence; one all of whose scores are -inf or NaN gives NaN.  scale: 1 / sqrt(D) if not given.

    Any row and head strides (copied where they are not multiples of 16 bytes).  Differentiable in q, k
    and v, once: a gradient of a gradient is an error.  What is not finite in one sequence, or behind the last
    one, changes nothing in another; within a sequence it may reach every query of the sequence, as in a product
    with a zero probability.

    The probabilities are rounded to the inputs' type for the product with v.  With a gradient to take, the result is
    divided by the sum of those rounded ones and its keys are not divided among SMs, without one (inference,
    ``no_grad``) it is the exact sum and they may be: the two differ by roundings, so a block that is recomputed
    for its backward pass does not repeat the bits of its first pass under ``no_grad``."""
    return _lib.torch_ops().packed_attention(q, k, v, offsets, k_offsets, causal, scale)


__all__ = ["packed_attention"]
