"""Gradients of rows whose weights are equal (queries of zeros, keys that repeat): o is then a mean of a few
bf16 values, which often lies in the very middle between two bf16 numbers.

With n equal scores every p is 1 before the division and the sums are n, both without rounding (a score's
exponent is off by 2^-19 at most for scores below 16).  What is left:
  o:      a sum of n values and a division, fp32, then kept to 2^-8 of bf16's last place, 2^-15 |o|
  delta:  2^-15 sum |do o| and the rounding of its D fp32 sums, D 2^-24 sum |do| |v|
  ds = p (dp - delta): those times p, dp's D sums, 2^-18 of itself for p, and half a bf16 step
  dq, dk: scale sum ds k, scale sum ds q; half a bf16 step of the result."""
import pytest
import torch

from prism_b200 import packed_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("keys", [2, 3, 4, 8])
@pytest.mark.parametrize("kind", ["zero queries", "repeated keys"])
@pytest.mark.parametrize("group", [1, 4])
def test_gradients_of_equal_weights(D, keys, kind, group, cuda):
    u, count, scale = 2.0 ** -8, 200, D ** -0.5
    g = torch.Generator(device="cuda").manual_seed(keys + D)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda").bfloat16()
    q, k, v, do = rnd(count, group, D), rnd(count * keys, 1, D), rnd(count * keys, 1, D), rnd(count, group, D)
    if kind == "zero queries":
        q.zero_()
    else:
        k = k.view(count, keys, 1, D)[:, :1].expand(-1, keys, -1, -1).reshape(count * keys, 1, D).contiguous()
    leaves = [t.requires_grad_() for t in (q, k, v)]
    at = torch.arange(count + 1, dtype=torch.int32, device="cuda")
    o = packed_attention(*leaves, at, at * keys, causal=False)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)

    Q, DO = (t.detach().double() for t in (q, do))                                   # [count, group, D]
    K, V = (t.detach().double().view(count, keys, D) for t in (k, v))
    mean = V.mean(1, keepdim=True)                                                   # o of every row
    dp, delta = DO @ V.transpose(1, 2), (DO * mean).sum(-1, keepdim=True)
    ds = (dp - delta) / keys
    sums = D * 2.0 ** -24 * (DO.abs() @ V.abs().transpose(1, 2))
    off = (sums + sums.mean(-1, keepdim=True) + 2.0 ** -15 * (DO * mean).abs().sum(-1, keepdim=True)) / keys
    off = off + (2.0 ** -18 + u) * (ds.abs() + off)
    assert bool(((o.detach().double() - mean).abs() <= (u + 2.0 ** -18) * mean.abs() + 2.0 ** -22 * V.abs().amax()).all())
    for got, ref, bound in ((dq, ds @ K * scale, off @ K.abs() * scale),
                            (dk, ds.transpose(1, 2) @ Q * scale, off.transpose(1, 2) @ Q.abs() * scale)):
        over = (got.double().view(ref.shape) - ref).abs() - bound - u * (ref.abs() + bound)
        assert bool((over <= 1e-30).all()), float((over / (bound + 1e-30)).max())
    # dv = sum over the group of p do; p = 1 / keys rounded once
    assert bool(((dv.double().view(V.shape) - (DO.sum(1, keepdim=True) / keys)).abs()
                 <= (2 * u + 2.0 ** -18) * 1.01 * DO.abs().sum(1, keepdim=True) / keys).all())
