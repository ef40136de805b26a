"""A paged cache (prism_b200.append_paged, paged_attention) against its definitions in float64.

Append: places and values bit for bit where nothing is rotated; rotated values within the bound of
apply_rotary's tests (1e-6 scale (|a| + |b|) for a pair (a, b), plus the output's rounding).
Attention: with u the rounding of the 16-bit type, p is rounded once for the product with v and the result once:
(u + 2e-4) sum_j p |v| + u |o|, the 2e-4 for all that is in fp32, as for packed_attention."""
import math

import pytest
import torch

from prism_b200 import _lib, append_paged, apply_rotary, packed_attention, paged_attention, rotary_frequencies

pytestmark = pytest.mark.gpu

RND = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}


class Cache:
    """Pages in a random order, a few unused, everything filled with `fill`."""

    def __init__(self, lengths, page, hk, D, dtype, fill=None, seed=0, spare=0, heads_first=False):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lengths]
        self.pages, self.page = sum(need) + 2, page
        order = torch.randperm(self.pages, generator=g).tolist()
        width = max(need + [1]) + spare
        rows, at = [], 0
        for n in need:
            rows.append(order[at:at + n] + [-7] * (width - n))
            at += n
        self.rows = rows
        self.table = torch.tensor(rows, dtype=torch.int32, device="cuda")
        gg = torch.Generator(device="cuda").manual_seed(seed)

        def make():
            shape = (self.pages, hk, page, D) if heads_first else (self.pages, page, hk, D)
            t = torch.randn(shape, generator=gg, device="cuda").to(dtype) if fill is None else torch.full(
                shape, fill, dtype=dtype, device="cuda")
            return t.transpose(1, 2) if heads_first else t

        self.k, self.v = make(), make()
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def where(self, b, token):
        return self.rows[b][token // self.page], token % self.page

    def tokens(self, cache, b, n):
        """The first n tokens of sequence b, [n, Hk, D]."""
        pages = torch.tensor(self.rows[b][:-(-n // self.page)], device="cuda", dtype=torch.long)
        return cache[pages].flatten(0, 1)[:n]


def _turned(x, positions, freqs, layout, scale):
    """float64, and |a| + |b| of each column's pair (0 for copied columns); x [T, H, D]."""
    x = x.double()
    rot = 2 * len(freqs)
    angle = positions.double()[:, None, None] * freqs
    pick = (lambda t: (t[..., 0:rot:2], t[..., 1:rot:2])) if layout == "interleaved" else \
        (lambda t: (t[..., :rot // 2], t[..., rot // 2:rot]))
    a, b = pick(x)
    out, size = x.clone(), torch.zeros_like(x)
    for half, y in zip(pick(out), (a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos())):
        half.copy_(y * scale)
    for half in pick(size):
        half.copy_((a.abs() + b.abs()) * scale)
    return out, size


def _check_turned(got, x, positions, freqs, layout, scale, what):
    ref, size = _turned(x, positions, freqs, layout, scale)
    bound = RND[got.dtype] * ref.abs() * 1.01 + 1e-6 * size + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    assert bool(((got.double() - ref).abs() <= bound).all()), what
    assert torch.equal(got[..., 2 * len(freqs):], x[..., 2 * len(freqs):]), what


def _append_case(new, before, hq, hk, D, rot, layout, page, dtype, form, strided=False, heads_first=False, wide=False):
    lengths = [a + b for a, b in zip(new, before)]
    c = Cache(lengths, page, hk, D, dtype, heads_first=heads_first)
    T = sum(new)
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(T, hq + 2 * hk, D + (8 if strided else 0), generator=g, device="cuda").to(dtype)[..., :D]
    q, k, v = qkv.split([hq, hk, hk], 1)
    if strided:   # the values' tokens are a head apart, their heads far
        v = v.transpose(0, 1).contiguous().transpose(0, 1)
    freqs = rotary_frequencies(rot, device="cuda")[0] if rot else None
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    offsets = torch.tensor(starts, dtype=torch.int64 if wide else torch.int32, device="cuda") if form == "packed" else None
    shape = (lambda t: t.unflatten(0, (len(new), -1))) if form == "each" else (lambda t: t)
    old_k, old_v = c.k.clone(), c.v.clone()
    version = c.k._version
    out = append_paged(shape(k), shape(v), c.k, c.v, c.table, c.lengths, offsets, q=shape(q), freqs=freqs, layout=layout,
                       scale=1.5 if rot else 1.0)
    assert c.k._version > version and c.v._version > 0
    assert out.shape == shape(q).shape and out.is_contiguous()
    positions = torch.tensor([p for n, m in zip(new, before) for p in range(m, m + n)], device="cuda")
    at = [c.where(b, p) for b, (n, m) in enumerate(zip(new, before)) for p in range(m, m + n)]
    if T:
        page_at, place_at = (torch.tensor(x, device="cuda") for x in zip(*at))
        assert torch.equal(c.v[page_at, place_at], v)
        spec = (positions, freqs if rot else torch.zeros(0, dtype=torch.float64, device="cuda"), layout, 1.5)
        _check_turned(c.k[page_at, place_at], k, *spec, "k")
        _check_turned(out.view(T, hq, D), q, *spec, "q")
        old_k[page_at, place_at], old_v[page_at, place_at] = c.k[page_at, place_at], c.v[page_at, place_at]
    assert torch.equal(old_k, c.k) and torch.equal(old_v, c.v)   # nothing else was written


@pytest.mark.parametrize("hq,hk,D,rot", [(4, 2, 128, 128), (1, 1, 64, 64), (5, 1, 128, 96), (3, 3, 64, 0), (2, 1, 80, 36),
                                         (2, 2, 256, 256), (1, 1, 7, 6), (2, 1, 36, 34)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", list(RND))
def test_append(hq, hk, D, rot, layout, dtype, cuda):
    _append_case([1, 1, 1], [0, 16, 130_999], hq, hk, D, rot, layout, 16, dtype, "one")
    _append_case([4, 4], [3, 90], hq, hk, D, rot, layout, 5, dtype, "each")
    _append_case([30, 0, 1, 150], [0, 7, 40, 9], hq, hk, D, rot, layout, 16, dtype, "packed")


@pytest.mark.parametrize("page", [1, 3, 64, 1000])
def test_append_strides_and_pages(page, cuda):
    _append_case([70, 9], [5, 0], 6, 2, 128, 128, "half", page, torch.bfloat16, "packed", strided=True, wide=True)
    _append_case([70, 9], [5, 0], 6, 2, 128, 64, "interleaved", page, torch.bfloat16, "packed", heads_first=True)
    _append_case([400] * 9, [5] * 9, 8, 8, 64, 64, "half", page, torch.float16, "each")


def test_append_matches_apply_rotary(cuda):
    """The queries and keys are rotated as apply_rotary rotates them, bit for bit."""
    c = Cache([900], 32, 2, 128, torch.bfloat16)
    q, k, v = torch.randn(900, 8, 128, device="cuda").bfloat16().split([4, 2, 2], 1)
    freqs, gain = rotary_frequencies(128, scaling="yarn", factor=4.0, original_length=256, device="cuda")
    out = append_paged(k[None], v[None], c.k, c.v, c.table, c.lengths, q=q[None], freqs=freqs, layout="half", scale=gain)
    qr, kr = apply_rotary(q, k, torch.arange(900, device="cuda"), freqs, layout="half", scale=gain)
    assert torch.equal(out[0], qr) and torch.equal(c.tokens(c.k, 0, 900), kr)


def test_append_without_queries(cuda):
    c = Cache([3, 4], 16, 2, 64, torch.float16, fill=0.0)
    k, v = torch.randn(2, 2, 4, 64, device="cuda").half().split(2, 2)
    assert append_paged(k, v, c.k, c.v, c.table, c.lengths) is None
    assert torch.equal(c.tokens(c.k, 0, 3)[1:], k[0]) and torch.equal(c.tokens(c.v, 1, 4)[2:], v[1])


def test_append_empty_slots_and_wrong_pages(cuda):
    """Empty slots and tokens of no sequence write nothing, wrong pages write nothing and show as NaN."""
    hk, D = 1, 64
    c = Cache([16, 16, 16, 16, 16], 16, hk, D, torch.bfloat16)
    old_k, old_v = c.k.clone(), c.v.clone()
    c.table[1, 0], c.table[2, 0] = -1, c.pages
    lengths = torch.tensor([0, 1, 2, 17, 5], dtype=torch.int32, device="cuda")   # 17: behind the table
    q, k, v = torch.randn(5, 3, D, device="cuda").bfloat16().split(1, 1)
    out = append_paged(k, v, c.k, c.v, c.table, lengths, q=q)
    assert not out[0].any() and all(bool(out[b].isnan().all()) for b in (1, 2, 3)) and torch.equal(out[4], q[4])
    old_k[c.rows[4][0], 4], old_v[c.rows[4][0], 4] = k[4], v[4]
    assert torch.equal(c.k, old_k) and torch.equal(c.v, old_v)
    # offsets that leave rows out, in front and behind
    offsets = torch.tensor([1, 1, 2, 2, 2, 3], dtype=torch.int32, device="cuda")
    out = append_paged(k, v, c.k, c.v, c.table, torch.tensor([0, 1, 0, 0, 9], dtype=torch.int32, device="cuda"), offsets, q=q)
    assert not out[0].any() and bool(out[1].isnan().all()) and torch.equal(out[2], q[2]) and not out[3:].any()
    old_k[c.rows[4][0], 8], old_v[c.rows[4][0], 8] = k[2], v[2]
    assert torch.equal(c.k, old_k) and torch.equal(c.v, old_v)


# ------------------------------------------------------------------ attention
def _attend(q, c, lengths, n, scale):
    """o and its bound, float64; q [B, n, Hq, D]."""
    u = RND[q.dtype]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    group = q.shape[2] // c.k.shape[2]
    for b, m in enumerate(lengths):
        if m == 0:
            continue
        k, v = (c.tokens(t, b, m).double() for t in (c.k, c.v))
        see = torch.arange(m, device="cuda") <= torch.arange(n, device="cuda")[:, None] + (m - n)
        for h in range(q.shape[2]):
            s = (q[b, :, h].double() @ k[:, h // group].T * scale).masked_fill(~see, -math.inf)
            top = s.amax(1, keepdim=True)
            p = torch.where(top == -math.inf, torch.zeros_like(s), (s - top.clamp_min(-1e300)).exp())
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            out[b, :, h] = p @ v[:, h // group]
            bound[b, :, h] = (u + 2e-4) * (p @ v[:, h // group].abs())
    return out, 1.01 * (bound + u * out.abs()) + (2.0 ** -24 if u < 2.0 ** -9 else 0.0)


def _attention_case(lengths, n, hq, hk, D, page, dtype, scale=None, seed=0, spread=1.5, **kw):
    c = Cache(lengths, page, hk, D, dtype, seed=seed, **kw)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn(len(lengths), n, hq, D, generator=g, device="cuda").mul_(spread).to(dtype)
    got = paged_attention(q if n > 1 else q[:, 0], c.k, c.v, c.table, c.lengths, scale=scale).view(q.shape)
    ref, bound = _attend(q, c, lengths, n, scale or D ** -0.5)
    off = (got.double() - ref).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-300)).max())


LENGTHS = [[1], [16, 17, 0, 15], [63, 64, 65, 128, 129], [100, 1, 300, 512], [513, 2, 700], [5000], [0, 3000, 64, 0, 65, 1], [0, 0]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("hq,hk", [(4, 1), (3, 3), (16, 2), (20, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", list(RND))
def test_one_token(lengths, hq, hk, D, dtype, cuda):
    _attention_case(lengths, 1, hq, hk, D, 16, dtype, seed=sum(lengths))


@pytest.mark.parametrize("n", [2, 5, 17, 64])
@pytest.mark.parametrize("hq,hk,D", [(4, 4, 64), (8, 2, 128), (5, 1, 64)])
@pytest.mark.parametrize("lengths", [[1, 300, 64], [1000, 0, 70]], ids=str)
def test_several_tokens(n, hq, hk, D, lengths, cuda):
    """Fewer keys than queries too: the first queries have none."""
    _attention_case(lengths, n, hq, hk, D, 16, torch.bfloat16, seed=n)


@pytest.mark.parametrize("page", [1, 7, 64, 100, 4096])
@pytest.mark.parametrize("heads_first", [False, True])
def test_pages(page, heads_first, cuda):
    _attention_case([700, 33, 1500], 1, 8, 2, 128, page, torch.bfloat16, heads_first=heads_first, spare=3)
    _attention_case([200, 33], 2, 8, 2, 64, page, torch.float16, heads_first=heads_first)


def test_wide_scores_and_scale(cuda):
    """Scores that raise the maximum often; their fp32 errors grow with them (300 (2^-23 + 2^-17) < 0.0024)."""
    for dtype in RND:
        c = Cache([2000], 16, 1, 64, dtype, seed=3)
        q = torch.randn(1, 1, 4, 64, device="cuda").mul_(20).to(dtype)
        got = paged_attention(q[:, 0], c.k, c.v, c.table, c.lengths, scale=0.3)
        ref, bound = _attend(q, c, [2000], 1, 0.3)
        c.v = c.v.abs()
        weight, _ = _attend(q, c, [2000], 1, 0.3)
        assert bool(((got.double() - ref[:, 0]).abs() <= (bound + 2.4e-3 * weight)[:, 0]).all())


def test_uneven_batch(cuda):
    """Many short sequences, one long one; more sequences than a CTA has threads."""
    _attention_case([40] * 100 + [9000] + [0, 200] * 60, 1, 4, 2, 64, 16, torch.bfloat16)


def test_what_lies_behind_the_end_does_not_matter(cuda):
    for lengths in ([100, 37, 0], [700, 1, 1029]):
        c = Cache(lengths, 16, 2, 64, torch.bfloat16, fill=math.nan)
        g = torch.Generator(device="cuda").manual_seed(0)
        for b, n in enumerate(lengths):
            for t in range(n):
                page, place = c.where(b, t)
                c.k[page, place] = torch.randn(2, 64, generator=g, device="cuda").bfloat16()
                c.v[page, place] = torch.randn(2, 64, generator=g, device="cuda").bfloat16()
        q = torch.randn(3, 1, 4, 64, generator=g, device="cuda").bfloat16()
        got = paged_attention(q[:, 0], c.k, c.v, c.table, c.lengths)
        ref, bound = _attend(q, c, lengths, 1, 0.125)
        assert bool(((got.double() - ref[:, 0]).abs() <= bound[:, 0]).all())


@pytest.mark.parametrize("page", [16, 256])   # without and with a divided grid
def test_wrong_pages_and_lengths_give_nan(page, cuda):
    c = Cache([3 * page] * 5, page, 1, 64, torch.bfloat16, spare=1)
    q = torch.randn(5, 2, 64, device="cuda").bfloat16()
    good = paged_attention(q, c.k, c.v, c.table, c.lengths)
    c.table[1, 1], c.table[2, 2] = -1, c.pages
    c.lengths[3] = 4 * page + 1
    c.lengths[4] = -3
    got = paged_attention(q, c.k, c.v, c.table, c.lengths)
    assert torch.equal(got[0], good[0]) and not got[4].any()
    assert all(bool(got[b].isnan().all()) for b in (1, 2, 3))


def test_no_table_and_no_cache(cuda):
    """A table without columns, a cache without pages: 0 without a token, NaN with one."""
    q = torch.randn(2, 2, 64, device="cuda").bfloat16()
    lengths = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    for pages, width in ((4, 0), (0, 1), (0, 0)):
        cache = [torch.zeros(pages, 16, 1, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
        table = torch.zeros(2, width, dtype=torch.int32, device="cuda")
        o = paged_attention(q, *cache, table, lengths)
        assert not o[0].any() and bool(o[1].isnan().all())
        new = torch.ones(2, 1, 64, device="cuda", dtype=torch.bfloat16)
        out = append_paged(new, new, *cache, table, lengths, q=q)
        assert not out[0].any() and bool(out[1].isnan().all()) and not cache[0].any()


def test_strided_queries(cuda):
    c = Cache([600, 40], 16, 2, 64, torch.bfloat16)
    qkv = torch.randn(2, 12, 64, device="cuda").bfloat16()
    for q in (qkv[:, :4], qkv[:, 2:12:2][:, :4], torch.randn(2, 4, 65, device="cuda").bfloat16()[..., 1:]):
        assert torch.equal(paged_attention(q, c.k, c.v, c.table, c.lengths),
                           paged_attention(q.contiguous(), c.k, c.v, c.table, c.lengths))


def test_far_places(cuda):
    """Elements past 2^31 of a cache."""
    pages, page, hk, D = 17000, 64, 16, 128     # 2.2e9 elements each
    k, v = (torch.zeros(pages, page, hk, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.tensor([[16999, 3, 16998]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([130], dtype=torch.int32, device="cuda")
    new = torch.randn(130, 3 * hk, D, device="cuda").bfloat16()
    q, kk, vv = new.split(hk, 1)
    append_paged(kk[None], vv[None], k, v, table, lengths)
    assert torch.equal(k[16999], kk[:64]) and torch.equal(v[16998, :2], vv[128:])
    c = Cache([130], page, hk, D, torch.bfloat16)
    c.k[c.rows[0]], c.v[c.rows[0]] = k[table[0].long()], v[table[0].long()]
    assert torch.equal(paged_attention(q[-1:], k, v, table, lengths), paged_attention(q[-1:], c.k, c.v, c.table, c.lengths))


def test_a_run(cuda):
    """Prompts through the packed attention, their keys and values to the cache, then tokens one by one, in a
    captured step: each token's output is that of packed attention over the whole sequence."""
    prompts, hq, hk, D, page, more = [37, 600, 1], 8, 2, 64, 16, 5
    total = [n + more for n in prompts]
    g = torch.Generator(device="cuda").manual_seed(2)
    raw = [torch.randn(n, hq + 2 * hk, D, generator=g, device="cuda").bfloat16() for n in total]
    freqs, _ = rotary_frequencies(D, device="cuda")
    whole = []
    for x in raw:
        q, k, v = x.split([hq, hk, hk], 1)
        q, k = apply_rotary(q, k, torch.arange(len(x), device="cuda"), freqs, layout="half")
        whole.append(packed_attention(q, k, v, torch.tensor([0, len(x)], dtype=torch.int32, device="cuda")))

    c = Cache(total, page, hk, D, torch.bfloat16, fill=math.nan)
    offsets = torch.tensor([0, 37, 637, 638], dtype=torch.int32, device="cuda")
    c.lengths.copy_(torch.tensor(prompts))
    q, k, v = torch.cat([x[:n] for x, n in zip(raw, prompts)]).split([hq, hk, hk], 1)
    q = append_paged(k, v, c.k, c.v, c.table, c.lengths, offsets, q=q, freqs=freqs, layout="half")
    kept = torch.cat([c.tokens(c.k, b, n) for b, n in enumerate(prompts)])
    o = packed_attention(q, kept, v, offsets)
    assert torch.equal(o, torch.cat([w[:n] for w, n in zip(whole, prompts)]))

    token = torch.empty(len(prompts), hq + 2 * hk, D, dtype=torch.bfloat16, device="cuda")

    def step():
        q, k, v = token.split([hq, hk, hk], 1)
        c.lengths.add_(1)
        q = append_paged(k, v, c.k, c.v, c.table, c.lengths, q=q, freqs=freqs, layout="half")
        return paged_attention(q, c.k, c.v, c.table, c.lengths)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    token.copy_(torch.stack([x[n] for x, n in zip(raw, prompts)]))
    with torch.cuda.stream(stream):
        first = step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    u = RND[torch.bfloat16]
    for i in range(more):
        if i:
            token.copy_(torch.stack([x[n + i] for x, n in zip(raw, prompts)]))
            graph.replay()
        got = first if i == 0 else out
        ref = torch.stack([w[n + i] for w, n in zip(whole, prompts)]).double()
        # both round p and the result: twice (u + 2e-4) sum p |v| + u |o|, |v| below 5 here
        top = max(float(x[:, hq + hk:].abs().max()) for x in raw)
        assert bool(((got.double() - ref).abs() <= 2 * (2 * u + 2e-4) * top).all())
    assert c.lengths.tolist() == total


def test_two_streams_and_two_graphs(cuda):
    """Calls that run at the same time, and two captured graphs replayed in turn, do not share a workspace."""
    cases = []
    for seed in (0, 1):
        c = Cache([3000, 50, 900], 16, 2, 128, torch.bfloat16, seed=seed)
        q = torch.randn(3, 8, 128, device="cuda").bfloat16()
        cases.append((c, q, paged_attention(q, c.k, c.v, c.table, c.lengths)))
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            c, q, _ = cases[i]
            with torch.cuda.stream(s):
                got[i].append(paged_attention(q, c.k, c.v, c.table, c.lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(x, cases[i][2]) for i in (0, 1) for x in got[i])
    graphs, outs = [], []
    for c, q, _ in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(paged_attention(q, c.k, c.v, c.table, c.lengths))
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, c[2]) for o, c in zip(outs, cases))


def test_gradients_are_refused(cuda):
    c = Cache([3], 16, 1, 64, torch.bfloat16)
    x = torch.randn(1, 1, 64, device="cuda").bfloat16().requires_grad_()
    with pytest.raises(NotImplementedError, match="inference only"):
        append_paged(x, x, c.k, c.v, c.table, c.lengths)
    with pytest.raises(NotImplementedError, match="inference only"):
        paged_attention(x, c.k, c.v, c.table, c.lengths)
    with torch.no_grad():
        paged_attention(x, c.k, c.v, c.table, c.lengths)
    assert _lib.load().prism_device_status() == 0
