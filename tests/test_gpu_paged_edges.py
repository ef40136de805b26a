"""paged_attention where new tokens have no key, or scores that the softmax leaves undefined."""
import math

import pytest
import torch

from prism_b200 import paged_attention

pytestmark = pytest.mark.gpu


def _cache(sequences, width, page, hk, D, dtype=torch.bfloat16):
    pages = sequences * width
    k, v = (torch.randn(pages, page, hk, D, device="cuda").to(dtype) for _ in "kv")
    order = torch.randperm(pages, device="cuda").to(torch.int32)
    return k, v, order.view(sequences, width)


@pytest.mark.parametrize("width", [4, 40])   # one launch, and shares that are joined
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("hq,hk", [(2, 2), (8, 2)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_new_tokens_without_keys(width, D, hq, hk, bad, cuda):
    """Fewer keys than new tokens: the first ones have none and give 0, whatever the values hold."""
    n, lengths = 6, [1, 4, 0, 600 if width == 40 else 30]
    k, v, table = _cache(4, width, 16, hk, D)
    for b, m in enumerate(lengths):
        if m:   # the newest token's value
            v[table[b, (m - 1) // 16], (m - 1) % 16] = bad
    q = torch.randn(4, n, hq, D, device="cuda").bfloat16()
    at = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    o = paged_attention(q, k, v, table, at)
    assert not o[0, :5].any() and not o[1, :2].any() and not o[2].any()
    assert not bool(o[[0, 1, 3], -1].isfinite().any())


@pytest.mark.parametrize("keys", [1, 20, 64, 200, 3000])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_that_are_not_finite(keys, D, dtype, cuda):
    """A query that is NaN, and one all of whose scores are -inf, give NaN; the others are as they were."""
    width = -(-keys // 16)
    k, v, table = _cache(4, width, 16, 1, D, dtype)
    k.abs_().add_(0.5)
    q = torch.rand(4, 2, D, device="cuda").to(dtype)
    at = torch.tensor([keys] * 4, dtype=torch.int32, device="cuda")
    want = paged_attention(q, k, v, table, at)
    q[1, 0], q[2, 1] = math.nan, -math.inf
    got = paged_attention(q, k, v, table, at)
    assert bool(got[1, 0].isnan().all()) and bool(got[2, 1].isnan().all())
    got[1, 0], got[2, 1] = want[1, 0], want[2, 1]
    assert torch.equal(got, want)
