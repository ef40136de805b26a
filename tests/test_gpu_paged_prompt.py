"""A prompt whose keys go to the cache attends itself with the keys of apply_rotary: the same bits as with those
that append_paged wrote, and the first answered token continues it."""
import pytest
import torch

from prism_b200 import append_paged, apply_rotary, packed_attention, paged_attention, rotary_frequencies

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_prompts_and_their_first_token(D, layout, cuda):
    prompts, hq, hk, page, width = [70, 1, 333], 8, 2, 16, 24
    g = torch.Generator(device="cuda").manual_seed(D)
    freqs, gain = rotary_frequencies(D, device="cuda")
    starts = [0, 70, 71, 404]
    offsets = torch.tensor(starts, dtype=torch.int32, device="cuda")
    lengths = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    caches = [torch.zeros(3 * width, page, hk, D, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    table = torch.randperm(3 * width, generator=g, device="cuda").to(torch.int32).view(3, width)
    positions = torch.cat([torch.arange(n, device="cuda") for n in prompts])
    rows = lambda n: torch.randn(n, hq + 2 * hk, D, generator=g, device="cuda").bfloat16().split([hq, hk, hk], 1)
    q, k, v = rows(starts[-1])
    turned = append_paged(k, v, *caches, table, lengths, offsets, q=q, freqs=freqs, layout=layout, scale=gain)
    also, keys = apply_rotary(q, k, positions, freqs, layout=layout, scale=gain)
    assert torch.equal(turned, also)
    kept = torch.cat([caches[0][table[b].long()].flatten(0, 1)[:n] for b, n in enumerate(prompts)])
    assert torch.equal(kept, keys)
    o = packed_attention(turned, keys, v, offsets)
    # the last token of each prompt by both ways: p rounded once or not, and each result: |v| below 6 here
    last = [e - 1 for e in starts[1:]]
    u = 2.0 ** -8
    by_page = paged_attention(turned[last], *caches, table, lengths)
    assert bool(((by_page.double() - o[last].double()).abs() <= (3 * u + 4e-4) * 6).all())
    # one more token each
    q1, k1, v1 = rows(3)
    lengths += 1
    got = paged_attention(append_paged(k1, v1, *caches, table, lengths, q=q1, freqs=freqs, layout=layout, scale=gain),
                          *caches, table, lengths)
    for b, n in enumerate(prompts):
        at = torch.full((1,), n, device="cuda")
        qb, kb = apply_rotary(q1[b:b + 1], k1[b:b + 1], at, freqs, layout=layout, scale=gain)
        K = torch.cat([keys[starts[b]:starts[b + 1]], kb]).double().repeat_interleave(hq // hk, 1)
        V = torch.cat([v[starts[b]:starts[b + 1]], v1[b:b + 1]]).double().repeat_interleave(hq // hk, 1)
        p = (torch.einsum("hd,mhd->hm", qb[0].double(), K) * D ** -0.5).softmax(-1)
        ref, weight = torch.einsum("hm,mhd->hd", p, V), torch.einsum("hm,mhd->hd", p, V.abs())
        assert bool(((got[b].double() - ref).abs() <= 1.01 * ((u * u + 2e-4) * weight + u * ref.abs())).all())
