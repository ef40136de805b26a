"""paged_attention's probabilities are held in two 16-bit parts: what is left of a p is u^2 of it, so that a
result is off by (u^2 + 2e-4) sum_j p |v| + u |o| (2e-4 for all that is in fp32, as in the other tests), where a p
rounded once would allow u sum_j p |v| more.  A row's largest p is no power of two here: its key lies tiles behind
the one that gave the running maximum, and less than 2^7 above it."""
import pytest
import torch

from prism_b200 import paged_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("keys", [400, 3000])   # one launch, and shares that are joined
def test_rows_with_one_dominant_key(dtype, D, keys, cuda):
    u, sequences, hk, group, page, scale = torch.finfo(dtype).eps / 2, 24, 2, 8, 16, 0.125
    g = torch.Generator(device="cuda").manual_seed(keys + D)
    width = keys // page + 1
    k, v = (torch.randn(sequences * width, page, hk, D, generator=g, device="cuda") for _ in "kv")
    k.mul_(0.1)
    table = torch.randperm(sequences * width, generator=g, device="cuda").to(torch.int32).view(sequences, width)
    q = torch.randn(sequences, hk * group, D, generator=g, device="cuda")
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    # of the first tile's four parts (16 keys each at 128 columns, 32 at 64) one key with a score of 6, most others 0
    for at in range(4, 4 * 2048 // D, 2048 // D):
        k[table[:, at // page].long(), at % page, :, 0] = 6.0
    at = 200   # and one of 7.5 to 10.8, e^1.5 to e^4.8 = 2^2.2 to 2^6.9 above those
    k[table[:, at // page].long(), at % page, :, 0] = 7.5 + 3.3 * torch.rand(sequences, hk, generator=g, device="cuda")
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    lengths = torch.full((sequences,), keys, dtype=torch.int32, device="cuda")
    got = paged_attention(q, k, v, table, lengths, scale=scale).double().unflatten(1, (hk, group))
    K, V = (t[table.long()].flatten(1, 2)[:, :keys].double().transpose(1, 2) for t in (k, v))   # [sequences, hk, keys, D]
    p = (q.double().unflatten(1, (hk, group)) @ K.transpose(2, 3) * scale).softmax(-1)
    o, weight = p @ V, p @ V.abs()
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    off = (got - o).abs()
    bound = 1.01 * ((u * u + 2e-4) * weight + u * o.abs()) + tiny
    assert bool((off <= bound).all()), float((off / bound).max())
