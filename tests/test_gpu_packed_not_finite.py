"""What the softmax leaves undefined is NaN and not the 0 of a row without keys: a query that is NaN, and scores
that are all -inf, wherever the mask leaves part of a half step (64 keys)."""
import math

import pytest
import torch

from prism_b200 import packed_attention

pytestmark = pytest.mark.gpu


def _at(*lists):
    return [torch.tensor(a, dtype=torch.int32, device="cuda") for a in lists]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,train", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float16, False)])
@pytest.mark.parametrize("row", [0, 5, 63, 64, 70])
@pytest.mark.parametrize("causal", [True, False])
def test_a_query_that_is_nan(D, dtype, train, row, causal, cuda):
    lengths = [80, 3, 40]
    starts = [0, 80, 83, 123]
    q, k, v = (torch.randn(123, h, D, device="cuda").to(dtype) for h in (4, 2, 2))
    at = _at(starts)[0]
    want = packed_attention(q, k, v, at, causal=causal)
    rows = [row, 80 + row % 3, 83 + row % 40]
    q[rows, 1] = math.nan
    leaves = [t.requires_grad_(train) for t in (q, k, v)]
    got = packed_attention(*leaves, at, causal=causal)
    assert bool(got[rows, 1].isnan().all())
    if not train:   # a query's scores are its own
        got[rows, 1] = want[rows, 1]
        assert torch.equal(got, want)
        return
    dq = torch.autograd.grad(got, leaves, torch.ones_like(got))[0]
    assert bool(dq[rows, 1].isnan().all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,train", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float16, False)])
@pytest.mark.parametrize("keys", [1, 60, 64, 100, 128, 200, 5000])
def test_scores_that_are_all_infinite(D, dtype, train, keys, cuda):
    """All scores of a query -inf: its softmax is 0 / 0.  5,000 keys are divided for inference."""
    q = torch.rand(10, 2, D, device="cuda").to(dtype)
    k, v = (torch.rand(keys, 1, D, device="cuda").add_(0.5).to(dtype) for _ in "kv")
    at = _at([0, 10], [0, keys])
    want = packed_attention(q, k, v, *at, causal=False)
    q[4] = -math.inf
    leaves = [t.requires_grad_(train) for t in (q, k, v)]
    got = packed_attention(*leaves, *at, causal=False)
    assert bool(got[4].isnan().all())
    if train:
        dq = torch.autograd.grad(got, leaves, torch.ones_like(got))[0]
        assert bool(dq[4].isnan().all())
    else:
        got[4] = want[4]
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,train", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float16, False)])
@pytest.mark.parametrize("keys", [100, 5000])
def test_some_scores_that_are_infinite(dtype, train, keys, cuda):
    """Keys at -inf, a whole step of them in front too, have no weight."""
    q = torch.rand(10, 2, 64, device="cuda").to(dtype)
    k, v = (torch.rand(keys, 1, 64, device="cuda").add_(0.5).to(dtype) for _ in "kv")
    k[:70] = -math.inf
    leaves = [t.requires_grad_(train) for t in (q, k, v)]
    got = packed_attention(*leaves, *_at([0, 10], [0, keys]), causal=False)
    ref = torch.softmax(q.detach().double().transpose(0, 1) @ k[70:, 0].detach().double().T * 0.125, -1) @ v[70:, 0].detach().double()
    u = torch.finfo(dtype).eps / 2
    # values between 0.5 and 1.5: half a step of p and one of the result, 2e-4 for what is in fp32
    assert bool(((got.detach().double().transpose(0, 1) - ref).abs() <= (2 * u + 2e-4) * 1.5).all())


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("n,m", [(300, 40), (2600, 2500)])
def test_rows_without_keys_stay_zero(train, n, m, cuda):
    """Also where their queries are not finite."""
    q, k, v = (torch.randn(r, h, 64, device="cuda").bfloat16() for r, h in ((n, 2), (m, 1), (m, 1)))
    q[: n - m] = math.nan
    leaves = [t.requires_grad_(train) for t in (q, k, v)]
    got = packed_attention(*leaves, *_at([0, n], [0, m]))
    assert not got[: n - m].any() and bool(got[n - m:].isfinite().all())
    if train:
        dq = torch.autograd.grad(got, leaves, torch.ones_like(got))[0]
        assert not dq[: n - m].any()
