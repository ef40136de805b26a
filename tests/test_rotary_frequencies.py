"""YaRN-scaled rotary frequencies at original lengths on both sides of every limit (no GPU needed).

Definition, with p(beta) the real pair index that turns beta times over the original length L,
p(beta) = rotary_dim ln(L / (2 pi beta)) / (2 ln theta): the ramp rises linearly from 0 at
floor(p(beta_fast)) to 1 at ceil(p(beta_slow)), and a pair's frequency is multiplied by
1 - ramp + ramp / factor.  The ramp's ends stay within [0, rotary_dim - 1]."""
import math

import pytest
import torch

from prism_b200.rotary import rotary_frequencies


def _ratio(rotary_dim, theta, factor, length, fast=32.0, slow=1.0):
    f, _ = rotary_frequencies(rotary_dim, theta)
    g, _ = rotary_frequencies(rotary_dim, theta, scaling="yarn", factor=factor, original_length=length, beta_fast=fast,
                              beta_slow=slow)
    return f * length / (2 * math.pi), (g / f).tolist()


@pytest.mark.parametrize("rotary_dim", [32, 64, 96, 128])
@pytest.mark.parametrize("theta", [1e4, 5e5])
@pytest.mark.parametrize("length", [2048, 4096, 32768, 65536, 131072, 1 << 20])
@pytest.mark.parametrize("factor", [4.0, 8.0])
def test_ramp_is_the_definitions(rotary_dim, theta, length, factor):
    _, ratio = _ratio(rotary_dim, theta, factor, length)
    p = lambda beta: rotary_dim * math.log(length / (2 * math.pi * beta)) / (2 * math.log(theta))
    low, high = max(math.floor(p(32.0)), 0), min(math.ceil(p(1.0)), rotary_dim - 1)
    for j, r in enumerate(ratio):
        ramp = min(max((j - low) / (high - low), 0.0), 1.0)
        assert math.isclose(r, 1 - ramp + ramp / factor, rel_tol=1e-12), (j, r)


@pytest.mark.parametrize("rotary_dim,length,factor", [(128, 65536, 4.0), (128, 131072, 8.0), (32, 65536, 4.0)])
def test_a_slowest_pair_that_turns_is_not_divided_by_the_whole_factor(rotary_dim, length, factor):
    turns, ratio = _ratio(rotary_dim, 1e4, factor, length)
    assert float(turns[-1]) > 1.2 and 1 / factor * 1.01 < ratio[-1] < 1


@pytest.mark.parametrize("length,slow", [(1, 1.0), (4, 1.0), (6, 1.0), (20, 4.0)])
def test_where_even_the_fastest_pair_turns_less_than_beta_slow(length, slow):
    """Every pair is divided by the factor, the first one too."""
    turns, ratio = _ratio(64, 1e4, 4.0, length, slow=slow)
    assert float(turns[0]) < slow
    assert all(math.isclose(r, 0.25, rel_tol=1e-12) for r in ratio)
