"""A sequence's bits do not depend on the rows behind it: those of the next sequence, or of no sequence, that
lie in its last tile.  Scores rise by 10 to 14 octaves from one half step (64 keys) to another, where a running
maximum may be kept or raised: the choice is the sequence's own."""
import math

import pytest
import torch

from prism_b200 import packed_attention

pytestmark = pytest.mark.gpu


def _rising(n, m, hq, hk, D, g):
    """n queries and m keys: column 0 makes chosen keys' scores rise, the other columns little."""
    q = torch.randn(n, hq, D, generator=g, device="cuda") * 0.3
    k = torch.randn(m, hk, D, generator=g, device="cuda") * 0.3
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    for key, octaves in ((70, 10.3), (150, 11.9), (200, 12.7), (330, 13.8)):   # second, first, second, second half
        k[key::400, :, 0] = octaves * math.log(2.0) * D ** 0.5
    return q.bfloat16(), k.bfloat16()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 8])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("n,m", [(50, 400), (19, 5000)])   # 5,000 keys are divided for inference
def test_rows_behind_a_sequence_do_not_matter(D, group, causal, train, n, m, cuda):
    hk, behind = 2, 60
    hq = hk * group
    g = torch.Generator(device="cuda").manual_seed(D + group + n)
    q, k = _rising(n + behind, m + behind, hq, hk, D, g)
    v = torch.randn(m + behind, hk, D, generator=g, device="cuda").bfloat16()
    do = torch.randn(n + behind, hq, D, generator=g, device="cuda").bfloat16()

    def run(q, k, v, do, next_sequence):
        at = [[0, n, n + behind], [0, m, m + behind]] if next_sequence else [[0, n, n], [0, m, m]]
        at = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in at]
        if not train:
            return [packed_attention(q, k, v, *at, causal=causal)[:n]]
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = packed_attention(*leaves, *at, causal=causal)
        dq, dk, dv = torch.autograd.grad(o, leaves, do)
        return [o.detach()[:n], dq[:n], dk[:m], dv[:m]]

    for next_sequence in (True, False):
        calm = [t.clone() for t in (q, k, v, do)]
        for t, end in zip(calm, (n, m, m, n)):
            t[end:] = 0
        want = run(*calm, next_sequence)
        assert all(bool(t.isfinite().all()) for t in want)
        for other in (math.nan, math.inf, -math.inf, 1e4):
            loud = [t.clone() for t in calm]
            for t, end in zip(loud, (n, m, m, n)):
                t[end:] = other
            if other == 1e4:   # scores that rise and fall by thousands
                loud[0][n:, :, 1::2] = -other
                loud[1][m:] = torch.randn_like(loud[1][m:]) * other
            for a, b in zip(want, run(*loud, next_sequence)):
                assert torch.equal(a, b), (next_sequence, other, int((a != b).sum()))
