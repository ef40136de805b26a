"""Keys and values kept in pages, for answering token by token: a cache is two tensors
[pages, page_size, Hk, D], and a table says which pages hold a sequence's tokens, in order, so that sequences
grow without being moved.

* ``append_paged`` puts new keys and values (whole prompts or single tokens) into their places, with the
  rotary positions of ``prism_b200.rotary`` applied to the keys and the queries on the way;
* ``paged_attention`` attends the cache with one or a few new tokens a sequence.  A whole prompt attends
  itself with ``prism_b200.packed.packed_attention``.

Both take ``lengths``, the number of tokens of each sequence with the new ones counted, so that a decoding
step is lengths += 1, append, attend; lengths and the table stay on the device and may change between the
replays of a captured graph.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib


def append_paged(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor, offsets: Optional[torch.Tensor] = None, *,
                 q: Optional[torch.Tensor] = None, freqs: Optional[torch.Tensor] = None,
                 layout: str = "interleaved", scale: float = 1.0) -> Optional[torch.Tensor]:
    """Writes k and v into the caches; returns q rotated like k (None without q).

    k, v [B, Hk, D] (one new token a sequence), [B, n, Hk, D] (n each), or [T, Hk, D] with offsets, int32 or int64
    [B + 1]: the new tokens of sequence b are the rows offsets[b] .. offsets[b + 1] - 1.  q alike, with its own
    heads.  bf16 or fp16, any strides of token and head; D up to 256.
    k_cache, v_cache [pages, page_size, Hk, D], any strides with contiguous columns, no two places on the same
    memory; page_table int32 [B, pages of a sequence]: token j is at place j % page_size of page
    page_table[b, j // page_size].
    lengths int32 [B]: each sequence's tokens, the new ones counted.
    freqs float64, layout, scale: as for ``apply_rotary``; the position is the token's number in its
    sequence.  Without freqs nothing is rotated.

    A token whose number would be negative (lengths[b] = 0: an empty slot of a padded batch), or that no
    sequence holds, writes nothing and its q is 0.  One whose page is not in the table or not in the cache
    writes nothing and its q is NaN.  Two new tokens may not have the same place.  Inference only."""
    return _lib.torch_ops().append_paged(k, v, k_cache, v_cache, page_table, lengths, offsets, q, freqs, layout, scale)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: Optional[float] = None) -> torch.Tensor:
    """q [B, Hq, D], or [B, n, Hq, D] for the last n tokens of each sequence, over the caches of
    ``append_paged`` -> the same shape: softmax(scale q k^T) v, query i over the keys up to its own place,
    lengths[b] - n + i.  D is 64 or 128; Hq a multiple of Hk.  scale: 1 / sqrt(D) if not given.  The caches' rows start
    on 16 bytes; caches of 64 GiB and more are refused.

    Meant for few tokens: 16 rows (query, head of a group) at a time read the sequence's keys.  A query without a
    key (lengths[b] < n: the first ones) gives 0; a sequence that is longer than its table, or whose table names a
    page that is not in the cache, gives NaN.  Cache places behind a sequence's end are not read.  A value that is
    not finite may reach every query of its sequence that has a key, one that does not see it too, as in a product
    with a zero probability.  Inference only."""
    return _lib.torch_ops().paged_attention(q, k_cache, v_cache, page_table, lengths, scale)


__all__ = ["append_paged", "paged_attention"]
