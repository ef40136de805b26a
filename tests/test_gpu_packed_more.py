"""Packed attention where work is divided or overlaps: parts of a tile's keys, other streams and late inputs,
captured backward passes, forward-mode derivatives."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from prism_b200 import _lib, append_paged, packed_attention, paged_attention
from test_gpu_packed_attention import _close, _exact, _inputs

pytestmark = pytest.mark.gpu


def _offsets(*lists):
    return [torch.tensor(a, dtype=torch.int32, device="cuda") for a in lists]


def _parts(q, k, count):
    """Whether the forward divides the keys of these shapes."""
    return _lib.load().prism_packed_attention_workspace_bytes(q.shape[0], k.shape[0], count, q.shape[1], k.shape[1], q.shape[2]) > 0


@pytest.mark.parametrize("q_len,k_len", [([40], [5000]), ([1, 300, 7], [3000, 4000, 2999]), ([20, 0, 9], [4000, 4000, 0]),
                                         ([700, 5], [6000, 1]), ([600], [1300])])
@pytest.mark.parametrize("hq,hk,D", [(4, 1, 128), (10, 2, 64), (3, 3, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
def test_parts_of_long_keys(q_len, k_len, hq, hk, D, dtype, causal, cuda):
    q, k, v, _, qa, ka = _inputs(q_len, k_len, hq, hk, D, dtype, seed=sum(q_len), before=3, behind=150)
    assert _parts(q, k, len(q_len))
    o = packed_attention(q, k, v, *_offsets(qa, ka), causal=causal)
    ref, bound = _exact(q, k, v, qa, ka, causal, D ** -0.5)
    _close(o, ref["o"], bound["o"], "o")


def test_parts_of_more_queries_than_keys_see(cuda):
    """Rows without a key in tiles whose other rows have many."""
    q, k, v, _, qa, ka = _inputs([2600, 100], [2500, 2600], 2, 2, 64, torch.bfloat16)
    assert _parts(q, k, 2)
    o = packed_attention(q, k, v, *_offsets(qa, ka))
    ref, bound = _exact(q, k, v, qa, ka, True, 0.125)
    _close(o, ref["o"], bound["o"], "o")
    assert not o[:100].any()


def test_parts_and_bad_offsets(cuda):
    q, k, v, _, _, _ = _inputs([90], [5000], 2, 1, 64, torch.bfloat16)
    for at in ([0, 50, 40], [0, 50, 91]):
        assert bool(packed_attention(q, k, v, *_offsets(at, [0, 2000, 5000])).isnan().all())
    clean = packed_attention(q, k, v, *_offsets([0, 50, 90], [0, 2000, 5000]))
    k[2000:], v[2000:] = math.nan, math.inf
    assert torch.equal(packed_attention(q, k, v, *_offsets([0, 50, 90], [0, 2000, 5000]))[:50], clean[:50])


def test_queries_of_many_tiles_on_few_keys(cuda):
    """Few key tiles: the sums of dK and dV are divided over the query tiles, in parts that see nothing too."""
    for q_len, k_len, causal in (([4000], [100], False), ([4000], [130], True), ([3000, 1500], [0, 70], False)):
        q, k, v, do, qa, ka = _inputs(q_len, k_len, 4, 2, 64, torch.bfloat16, before=2, behind=40)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        o = packed_attention(*leaves, *_offsets(qa, ka), causal=causal)
        ref, bound = _exact(q.detach(), k.detach(), v.detach(), qa, ka, causal, 0.125, do)
        _close(o.detach(), ref["o"], bound["o"], "o")
        for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)):
            _close(t, ref[n], bound[n], n)


def test_items_of_all_sizes(cuda):
    """More tiles than the GPU has SMs, from one step to many, so that CTAs go from one to the next; odd lengths
    leave tails between them."""
    lengths = [1, 700, 33, 0, 1500, 129, 64, 900, 5, 257, 1100, 2] * 3
    for D, causal in ((64, True), (128, True), (64, False), (128, False)):
        q, k, v, do, qa, ka = _inputs(lengths, lengths, 8, 4, D, torch.bfloat16, seed=D)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        o = packed_attention(*leaves, _offsets(qa)[0], causal=causal)
        ref, bound = _exact(q.detach(), k.detach(), v.detach(), qa, ka, causal, D ** -0.5, do)
        _close(o.detach(), ref["o"], bound["o"], "o")
        for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)):
            _close(t, ref[n], bound[n], n)
    assert _lib.load().prism_device_status() == 0


def test_equal_scores(cuda):
    """All p alike and as large as a fresh maximum gives: within fp16."""
    for dtype in (torch.bfloat16, torch.float16):
        k = torch.randn(1000, 2, 64, device="cuda").to(dtype)
        q, at = torch.zeros_like(k), [0, 1000]
        o = packed_attention(q, k, k, _offsets(at)[0], causal=False)
        ref, bound = _exact(q, k, k, at, at, False, 0.125)
        _close(o, ref["o"], bound["o"], str(dtype))


def _both(q, k, v, do, offsets):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = packed_attention(*leaves, offsets)
    return [o.detach(), *torch.autograd.grad(o, leaves, do)]


def test_behind_late_inputs_on_another_stream(cuda):
    """A launch on any other stream than the current one would read zeros."""
    q, k, v, do, qa, _ = _inputs([300, 77], [300, 77], 4, 2, 64, torch.bfloat16)
    offsets, lengths, table = _offsets(qa, [300, 77], [[0, 1, 2, 3, 4], [5, 6, -1, -1, -1]])
    cache = lambda: [torch.zeros(7, 64, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]

    def run(q, k, v, do, offsets, lengths):
        pages = cache()
        turned = append_paged(k, v, *pages, table, lengths, offsets, q=q)
        return _both(q, k, v, do, offsets) + [turned, *pages, paged_attention(q[[299, 376]], *pages, table, lengths)]

    given = (q, k, v, do, offsets, lengths)
    want = run(*given)
    late = [torch.zeros_like(t) for t in given]
    busy = torch.randn(8192, 8192, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy @ busy
        for a, b in zip(late, given):
            a.copy_(b)
        got = run(*late)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once(cuda):
    """Calls that divide their work and run next to each other on two streams keep their workspaces apart."""
    cases = [_inputs([900, 40], [900, 40], 8, 2, D, torch.bfloat16, seed=D) for D in (64, 128)]
    long = [_inputs([60], [6000], 4, 1, D, torch.bfloat16, seed=D) for D in (64, 128)]

    def run(i):
        q, k, v, do, qa, _ = cases[i]
        lq, lk, lv, _, la, lka = long[i]
        return _both(q, k, v, do, at[i]) + [packed_attention(lq, lk, lv, *lat[i])]

    at, lat = [_offsets(c[4])[0] for c in cases], [_offsets(c[4], c[5]) for c in long]
    want = [run(0), run(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(a, b) for r in got[i] for a, b in zip(r, want[i]))


def test_captured_training_step(cuda):
    """Forward and backward in one graph, replayed with new values and lengths."""
    q, k, v, do, qa, _ = _inputs([100, 130], [100, 130], 4, 2, 64, torch.bfloat16)
    offsets = _offsets(qa)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _both(q, k, v, do, offsets)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _both(q, k, v, do, offsets)
    for at in ([0, 100, 230], [0, 7, 229], [0, 0, 230]):
        offsets.copy_(torch.tensor(at, dtype=torch.int32))
        q.mul_(0.75)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, _both(q, k, v, do, offsets)))


def test_first_call_of_a_thread(cuda):
    """A backward pass whose thread has called nothing before."""
    import threading
    q, k, v, do, qa, _ = _inputs([70], [70], 2, 1, 64, torch.bfloat16)
    offsets, got = _offsets(qa)[0], []
    want = _both(q, k, v, do, offsets)
    torch.cuda.synchronize()
    thread = threading.Thread(target=lambda: got.extend(_both(q, k, v, do, offsets)))
    thread.start(), thread.join()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_mode_is_refused(cuda):
    q, k, v, _, qa, _ = _inputs([40], [40], 2, 2, 64, torch.bfloat16)
    offsets = _offsets(qa)[0]
    cache = [torch.zeros(3, 16, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    table, lengths = _offsets([[0, 1, 2]], [40])
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: packed_attention(dual(q), k, v, offsets), lambda: packed_attention(q, dual(k), v, offsets),
                     lambda: packed_attention(q, k, dual(v), offsets), lambda: append_paged(dual(k)[None], v[None], *cache, table, lengths),
                     lambda: append_paged(k[None], v[None], *cache, table, lengths, q=dual(q)[None]),
                     lambda: paged_attention(dual(q)[:1], *cache, table, lengths),
                     lambda: paged_attention(q[:1], dual(cache[0]), cache[1], table, lengths)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_other_devices_are_refused(cuda):
    q, k, v, _, qa, _ = _inputs([40], [40], 2, 2, 64, torch.bfloat16)
    with pytest.raises(_lib.PrismError):
        packed_attention(q, k, v, torch.tensor(qa, dtype=torch.int32))
    cache = [torch.zeros(3, 16, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    table, lengths = _offsets([[0, 1, 2]], [40])
    with pytest.raises(_lib.PrismError):
        paged_attention(q[:1], *cache, table.cpu(), lengths)
    with pytest.raises(_lib.PrismError):
        append_paged(k[None], v[None], *cache, table, lengths.cpu())
    with pytest.raises(ValueError, match="16 bytes"):
        paged_attention(q[:1], *[torch.zeros(3 * 16 * 2 * 64 + 4, device="cuda", dtype=torch.bfloat16)[4:].view(3, 16, 2, 64)] * 2,
                        table, lengths)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group", [1, 8, 37])
def test_same_bits_many_times(D, group, cuda):
    """Warps that run ahead of others by as much as the barriers let them: the same bits every time."""
    q_len = [1, 0, 1100, 306, 700, 1, 0, 2010, 565, 44] * 2
    k_len = [600, 1800, 1400, 906, 2500, 0, 318, 2500, 1, 1212] * 2
    q, k, v, do, qa, ka = _inputs(q_len, k_len, group, 1, D, torch.bfloat16, seed=group)
    for causal in (True, False):
        leaves, at, first = [t.requires_grad_() for t in (q, k, v)], _offsets(qa, ka), None
        for _ in range(40):
            o = packed_attention(*leaves, *at, causal=causal)
            got = [o.detach(), *torch.autograd.grad(o, leaves, do)]
            first = first or got
            assert all(torch.equal(a, b) and not bool(a.isnan().any()) for a, b in zip(got, first))


@pytest.mark.parametrize("D,group", [(64, 1), (64, 4), (128, 1), (128, 8)])
def test_gradients_of_rows_with_one_dominant_key(D, group, cuda):
    """One query a sequence with most of its weight on one key: ds = p (do . v - delta) is a small difference.
    Element by element: half steps of 2^-8 (bf16) of o's weights, which move delta by 2^-8 of the sum of |ds|
    and once more in their sum; of ds and of p by as much of |ds|; of dq itself.  o is kept to 2^-15, and the fp32
    sums of up to 451 products to 451 2^-24 of their terms' magnitudes (in s: times the exponent's slope, |ds|)."""
    u, count, keys, scale = 2.0 ** -8, 48, 451, D ** -0.5
    q, k, v, do, qa, ka = _inputs([1] * count, [keys] * count, 2 * group, 2, D, torch.bfloat16, seed=D + group)
    q *= 6
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = packed_attention(*leaves, *_offsets(qa, ka))
    dq, dk = torch.autograd.grad(o, leaves[:2], do)
    rows, cols = slice(qa[0], qa[-1]), slice(ka[0], ka[-1])
    Q, DO = (t[rows].detach().double().unflatten(1, (2, group)) for t in (q, do))          # [count, 2, group, D]
    K, V = (t[cols].detach().double().unflatten(0, (count, keys)).transpose(1, 2) for t in (k, v))  # [count, 2, keys, D]
    p = (Q @ K.transpose(2, 3) * scale).softmax(-1)
    dp, delta = DO @ V.transpose(2, 3), (DO * (p @ V)).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    sums = keys * 2.0 ** -24
    off_s = sums * (Q.abs() @ K.abs().transpose(2, 3)) * scale
    terms = DO.abs() @ V.abs().transpose(2, 3)
    off = (2 * u + 2 * off_s.amax(-1, keepdim=True)) * ds.abs() + sums * p * terms
    off += p * (2 * u * ds.abs().sum(-1, keepdim=True) + 2.0 ** -15 * (DO * (p @ V)).abs().sum(-1, keepdim=True)
                + sums * (p * terms).sum(-1, keepdim=True))
    for got, ref, bound in ((dq[rows].double().unflatten(1, (2, group)), ds @ K * scale, off @ K.abs() * scale),
                            (dk[cols].double().unflatten(0, (count, keys)).transpose(1, 2), ds.transpose(2, 3) @ Q * scale,
                             off.transpose(2, 3) @ Q.abs() * scale)):
        assert bool(((got - ref).abs() <= bound + u * (ref.abs() + bound) + 1e-30).all())
