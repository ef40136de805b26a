"""Caches with dimensions of size one."""
import pytest
import torch

from prism_b200 import append_paged, paged_attention

pytestmark = pytest.mark.gpu


def _strided(shape, strides, dtype=torch.bfloat16):
    return torch.randn(1 << 16, device="cuda").to(dtype)[: 1 + sum((n - 1) * s for n, s in zip(shape, strides))].as_strided(shape, strides)


@pytest.mark.parametrize("shape,strides", [((4, 16, 1, 64), (1024, 64, 3, 1)), ((1, 32, 2, 64), (7, 128, 64, 1)),
                                           ((6, 1, 2, 64), (128, 5, 64, 1)), ((1, 1, 1, 64), (1, 1, 1, 1))])
def test_strides_of_dimensions_of_one(shape, strides, cuda):
    """The stride of a dimension of size one is never used, so that it may be anything."""
    k, v = _strided(shape, strides), _strided(shape, strides)
    pages, page, hk, D = shape
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    lengths = torch.tensor([pages * page], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4 * hk, D, device="cuda").bfloat16()
    plain = [t.clone(memory_format=torch.contiguous_format) for t in (k, v)]
    assert torch.equal(paged_attention(q, k, v, table, lengths), paged_attention(q, *plain, table, lengths))
    new = torch.randn(2, 1, hk, D, device="cuda").bfloat16()
    for cache in ((k, v), plain):
        append_paged(new[0], new[1], *cache, table, lengths)
    assert torch.equal(k, plain[0]) and torch.equal(v, plain[1])
