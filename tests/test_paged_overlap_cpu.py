"""append_paged writes into the caches: places that share memory are refused (no GPU needed)."""
import pytest
import torch

from prism_b200 import append_paged


def _call(k_cache, v_cache):
    new = torch.zeros(3, k_cache.shape[2], k_cache.shape[3], dtype=torch.bfloat16)
    table = torch.zeros(3, 2, dtype=torch.int32)
    append_paged(new, new, k_cache, v_cache, table, torch.ones(3, dtype=torch.int32))


def _cache(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("make", [
    lambda: _cache(1, 16, 2, 64).expand(4, -1, -1, -1),
    lambda: _cache(4, 1, 2, 64).expand(-1, 16, -1, -1),
    lambda: _cache(4, 16, 1, 64).expand(-1, -1, 2, -1),
    lambda: _cache(10000).as_strided((4, 16, 2, 64), (2048, 128, 32, 1)),    # heads half on each other
    lambda: _cache(10000).as_strided((4, 16, 2, 64), (1024, 128, 64, 1)),    # pages half on each other
])
def test_overlapping_places_are_refused(make):
    fine = _cache(4, 16, 2, 64)
    for caches in ((make(), fine), (fine, make())):
        with pytest.raises(ValueError, match="share memory"):
            _call(*caches)


def test_one_cache_for_both_is_refused():
    both = _cache(4, 16, 2, 64)
    with pytest.raises(ValueError, match="share memory"):
        _call(both, both)
    with pytest.raises(ValueError, match="share memory"):
        _call(both, both[:])


@pytest.mark.parametrize("make", [
    lambda: [_cache(4, 16, 2, 64), _cache(4, 16, 2, 64)],
    lambda: _cache(4, 2, 16, 2, 64).unbind(1),                       # keys and values of a page side by side
    lambda: _cache(4, 16, 2, 2, 64).unbind(2),
    lambda: _cache(4, 16, 2, 128).chunk(2, -1),
    lambda: [t.transpose(1, 2) for t in _cache(2, 4, 2, 16, 64)],    # heads first
    lambda: _cache(2, 4, 16, 1, 64).expand(2, 4, 16, 1, 64).unbind(0),
    lambda: [_cache(70000).as_strided((4, 16, 1, 64), (1024, 64, 0, 1)), _cache(4, 16, 1, 64)],   # a dimension of one
    lambda: [_cache(0, 16, 2, 64), _cache(0, 16, 2, 64)],
])
def test_other_caches_reach_the_device_check(make):
    from prism_b200 import _lib
    with pytest.raises(_lib.PrismError, match="CUDA"):
        _call(*make())
