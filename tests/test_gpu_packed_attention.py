"""Dense attention over packed sequences (prism_b200.packed_attention) against its formulas in float64.

Bounds, with u the rounding of the 16-bit type (eps / 2) and X = 2e-4 for everything in fp32: a score is off
by at most D 2^-24 sum |q k| scale and its exponent by another 2^-23 |s|, below 1e-4 for the inputs here, the
exponential and the sums add a few 2^-22.
  o:  p is rounded once for the product with v, the result once:  (u + X) sum_j p |v| + u |o|
  dv: likewise                                                    (u + X) sum_i p |do| + u |dv|
  ds = p (dp - delta): rounded once; delta is formed from the rounded o, so it is off by at most
      E_i = sum_d |do_d| bound(o_d) + X sum_d |do_d| max|v|:      |ds| (u + X) + p E_i
  dq, dk: scale sum bound(ds) |k| + u |dq|, scale sum bound(ds) |q| + u |dk|
times 1.01 for the second order."""
import math

import pytest
import torch

from prism_b200 import _lib, packed_attention

pytestmark = pytest.mark.gpu

X = 2e-4


def _starts(lengths, first=0):
    out = [first]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _exact(q, k, v, q_at, k_at, causal, scale, do=None):
    """o, dq, dk, dv and their bounds, float64; rows of no sequence 0 (bound 0)."""
    u = torch.finfo(q.dtype).eps / 2
    q, k, v = q.double(), k.double(), v.double()
    names = ["o"] + (["dq", "dk", "dv"] if do is not None else [])
    like = {"o": q, "dq": q, "dk": k, "dv": v}
    out = {n: torch.zeros_like(like[n]) for n in names}
    bound = {n: torch.zeros_like(like[n]) for n in names}
    group = q.shape[1] // k.shape[1]
    for b in range(len(q_at) - 1):
        r, c = slice(q_at[b], q_at[b + 1]), slice(k_at[b], k_at[b + 1])
        n, m = q_at[b + 1] - q_at[b], k_at[b + 1] - k_at[b]
        if n == 0 or m == 0:
            continue
        for h in range(q.shape[1]):
            qh, kh, vh = q[r, h], k[c, h // group], v[c, h // group]
            s = qh @ kh.T * scale
            if causal:
                s = s.masked_fill(torch.arange(m, device=q.device) > torch.arange(n, device=q.device)[:, None] + (m - n),
                                  -math.inf)
            top = s.amax(1, keepdim=True)
            p = torch.where(top == -math.inf, torch.zeros_like(s), (s - top.clamp_min(-1e300)).exp())
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            o = p @ vh
            bo = (u + X) * (p @ vh.abs()) + u * o.abs()
            out["o"][r, h], bound["o"][r, h] = o, bo
            if do is None:
                continue
            g = do[r, h].double()
            ds = p * (g @ vh.T - (g * o).sum(1, keepdim=True))
            far = (g.abs() * bo).sum(1, keepdim=True) + X * g.abs().sum(1, keepdim=True) * vh.abs().max()
            bds = ds.abs() * (u + X) + p * far
            out["dq"][r, h] = ds @ kh * scale
            bound["dq"][r, h] = bds @ kh.abs() * scale
            out["dk"][c, h // group] += ds.T @ qh * scale
            bound["dk"][c, h // group] += bds.T @ qh.abs() * scale
            out["dv"][c, h // group] += p.T @ g
            bound["dv"][c, h // group] += (u + X) * (p.T @ g.abs())
    for n in names[1:]:
        bound[n] += u * out[n].abs()
    tiny = 2.0 ** -24 if u < 2.0 ** -9 else 0.0   # fp16: half of its smallest number, for a result near 0
    return out, {n: 1.01 * t + tiny for n, t in bound.items()}


def _close(got, ref, bound, what):
    assert got.shape == ref.shape, what
    off = (got.double() - ref).abs()
    assert bool((off <= bound).all()), (what, float((off / bound.clamp_min(1e-300)).max()), off.flatten().argmax())


def _inputs(q_len, k_len, hq, hk, D, dtype, seed=0, before=0, behind=0, strided=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, Tk = before + sum(q_len) + behind, before + sum(k_len) + behind

    def rnd(n, heads):
        if strided:   # a slice of wider rows, heads outside of the rows
            return torch.randn(heads + 1, n, D + 8, generator=g, device="cuda").to(dtype)[1:, :, :D].transpose(0, 1)
        return torch.randn(n, heads, D, generator=g, device="cuda").to(dtype)

    return rnd(T, hq), rnd(Tk, hk), rnd(Tk, hk), rnd(T, hq), _starts(q_len, before), _starts(k_len, before)


def _run(q_len, k_len, hq, hk, D, causal, dtype=torch.bfloat16, grad=True, wide=False, scale=None, own_keys=None, **kw):
    q, k, v, do, qa, ka = _inputs(q_len, k_len, hq, hk, D, dtype, **kw)
    kind = torch.int64 if wide else torch.int32
    offsets, k_offsets = (torch.tensor(a, dtype=kind, device="cuda") for a in (qa, ka))
    for t in (q, k, v):
        t.requires_grad_(grad)
    o = packed_attention(q, k, v, offsets, None if own_keys is None and q_len == k_len else k_offsets, causal=causal,
                         scale=scale)
    ref, bound = _exact(q.detach(), k.detach(), v.detach(), qa, ka, causal, scale or D ** -0.5, do if grad else None)
    _close(o.detach(), ref["o"], bound["o"], "o")
    assert o.dtype == dtype and o.is_contiguous()
    if grad:
        for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)):
            _close(t, ref[n], bound[n], n)
    assert _lib.load().prism_device_status() == 0


LENGTHS = [[1], [2, 1, 3], [127], [128], [129], [64, 200, 1, 0, 255, 256, 257], [0, 0, 5, 0], [700], [1] * 40]


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("hq,hk", [(2, 2), (8, 2), (3, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_own_keys(lengths, hq, hk, D, causal, cuda):
    _run(lengths, lengths, hq, hk, D, causal, seed=len(lengths) + hq)


@pytest.mark.parametrize("q_len,k_len", [([1, 1, 1], [300, 1, 129]), ([5, 70, 130], [5, 200, 131]), ([40], [1000]),
                                         ([256, 3], [384, 128]), ([10, 20], [0, 7]), ([300], [40]), ([0, 9], [30, 9]),
                                         ([200, 129], [130, 1])])
@pytest.mark.parametrize("hq,hk,D", [(4, 1, 128), (2, 2, 64), (10, 2, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_other_keys(q_len, k_len, hq, hk, D, causal, cuda):
    """Queries at the end of their keys; with more queries than keys the first ones see none."""
    _run(q_len, k_len, hq, hk, D, causal, seed=sum(q_len))


@pytest.mark.parametrize("group", [1, 5, 7, 16, 33, 64, 100, 128])
def test_groups(group, cuda):
    """Groups that divide a tile's 128 rows and that leave some over."""
    _run([37, 150, 3], [37, 150, 3], group, 1, 64, True, seed=group)
    _run([21], [210], 2 * group, 2, 128, True, seed=group)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("spread", [1.0, 12.0])
def test_half_precision(D, causal, spread, cuda):
    """fp16 forward; with wide scores the running maximum is raised often."""
    q_len, k_len = [130, 1, 77], [700, 300, 77]
    q, k, v, _, qa, ka = _inputs(q_len, k_len, 4, 2, D, torch.float16, seed=3)
    q *= spread
    offsets, k_offsets = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in (qa, ka))
    o = packed_attention(q, k, v, offsets, k_offsets, causal=causal)
    # scores up to `spread` times as large: so is their error
    ref, bound = _exact(q, k, v, qa, ka, causal, D ** -0.5)
    _close(o, ref["o"], bound["o"] * (1 + (spread - 1) * X / (X + 2.0 ** -11)), "o")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rising_scores(dtype, cuda):
    """Keys whose scores rise by a lot from tile to tile (each step rescales) and one far above the rest."""
    n, D = 900, 128
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.ones(n, 1, D, device="cuda", dtype=dtype)
    k = (torch.arange(n, device="cuda")[:, None, None] / 8.0).expand(n, 1, D).to(dtype).contiguous() * 0.125
    v = torch.randn(n, 1, D, generator=g, device="cuda").to(dtype)
    at = [0, n]
    offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
    for flip in (False, True):
        kk = k.flip(0).contiguous() if flip else k
        o = packed_attention(q, kk, v, offsets)
        # scores up to 160: exponents are off by 160 (2^-23 + 128 2^-24), 0.0013 at most
        ref, bound = _exact(q, kk, v, at, at, True, D ** -0.5)
        weight = _exact(q, kk, v.abs(), at, at, True, D ** -0.5)[0]["o"]
        _close(o, ref["o"], bound["o"] + 1.4e-3 * weight, f"flip {flip}")


@pytest.mark.parametrize("causal", [True, False])
def test_strides_offsets_and_scale(causal, cuda):
    _run([65, 30, 190], [65, 30, 190], 6, 2, 64, causal, strided=True, wide=True, scale=0.3)
    _run([65, 30, 190], [33, 140, 1], 6, 3, 128, causal, strided=True, before=5, behind=300)
    _run([9], [9], 2, 1, 64, causal, before=130, behind=1)


def test_long_rows_many_sequences(cuda):
    """More sequences than a CTA has threads, and a long one between them."""
    lengths = [3] * 200 + [2000] + [1, 0, 5] * 100
    _run(lengths, lengths, 2, 1, 64, True, seed=9)


@pytest.mark.parametrize("D", [64, 128])
def test_other_sequences_do_not_matter(D, cuda):
    """A NaN or an infinity in the neighbours, before the first and behind the last one changes nothing."""
    q, k, v, do, qa, ka = _inputs([50, 77, 90], [40, 333, 20], 4, 2, D, torch.bfloat16, before=3, behind=70)
    offsets, k_offsets = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in (qa, ka))

    def run(a, b, c, d):
        a, b, c = (t.clone().requires_grad_() for t in (a, b, c))
        o = packed_attention(a, b, c, offsets, k_offsets, causal=causal)
        return [o.detach()] + list(torch.autograd.grad(o, (a, b, c), d))

    for causal in (True, False):
        clean = run(q, k, v, do)
        for bad in (math.nan, math.inf):
            dirty = [t.clone() for t in (q, k, v, do)]
            for t, at in zip(dirty, (qa, ka, ka, qa)):
                t[:at[1]] = bad
                t[at[2]:] = bad
            for a, b, at in zip(clean, run(*dirty), (qa, qa, ka, ka)):
                assert torch.equal(a[at[1]:at[2]], b[at[1]:at[2]])
                assert not b[:at[0]].any() and not b[at[3]:].any()


def test_gradient_against_differences(cuda):
    """The gradient along a direction, and the difference quotient of the formula in float64."""
    q, k, v, do, qa, ka = _inputs([100, 31], [100, 31], 4, 2, 64, torch.bfloat16, seed=4)
    offsets = torch.tensor(qa, dtype=torch.int32, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(packed_attention(*leaves, offsets), leaves, do)
    _, bound = _exact(q, k, v, qa, ka, True, 0.125, do)
    loss = lambda *t: float((_exact(*t, qa, ka, True, 0.125)[0]["o"] * do.double()).sum())
    g = torch.Generator(device="cuda").manual_seed(8)
    for i, name in enumerate(("dq", "dk", "dv")):
        base = [t.double() for t in (q, k, v)]
        way = torch.randn(base[i].shape, generator=g, device="cuda", dtype=torch.float64)
        step = 1e-5
        ends = []
        for sign in (1, -1):
            moved = list(base)
            moved[i] = base[i] + sign * step * way
            ends.append(loss(*moved))
        slope = (ends[0] - ends[1]) / (2 * step)
        # the quotient's own error: some step^2, and 1e-16 / step of the loss
        assert abs(float((grads[i].double() * way).sum()) - slope) <= float((bound[name] * way.abs()).sum()) + 1e-5


def test_parts_of_the_gradient(cuda):
    """Only some inputs require a gradient; the same values as with all of them."""
    q, k, v, do, qa, _ = _inputs([60, 130], [60, 130], 2, 2, 64, torch.bfloat16)
    offsets = torch.tensor(qa, dtype=torch.int32, device="cuda")
    full = [t.clone().requires_grad_() for t in (q, k, v)]
    all_of = torch.autograd.grad(packed_attention(*full, offsets), full, do)
    for i in range(3):
        some = [t.clone() for t in (q, k, v)]
        some[i].requires_grad_()
        assert torch.equal(torch.autograd.grad(packed_attention(*some, offsets), some[i], do)[0], all_of[i])
    # a gradient without strides of its own
    o = packed_attention(*full, offsets)
    a = torch.autograd.grad(o.float().sum(), full, retain_graph=True)
    b = torch.autograd.grad(o, full, torch.ones_like(o))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_same_bits_again(cuda):
    """Fixed summation orders: the same call gives the same bits, on another stream too."""
    q, k, v, do, qa, _ = _inputs([500, 3, 900], [500, 3, 900], 8, 2, 128, torch.bfloat16)
    offsets = torch.tensor(qa, dtype=torch.int32, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]

    def run():
        o = packed_attention(*leaves, offsets)
        return [o.detach()] + list(torch.autograd.grad(o, leaves, do))

    first = run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = run()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_captured(cuda):
    """Captured forward passes replay with new values and new offsets in the same buffers."""
    q, k, v, _, qa, _ = _inputs([100, 28], [100, 28], 4, 2, 64, torch.bfloat16)
    offsets = torch.tensor(qa, dtype=torch.int32, device="cuda")
    packed_attention(q, k, v, offsets)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = packed_attention(q, k, v, offsets)
    for at in ([0, 100, 128], [0, 1, 128], [0, 60, 61]):
        offsets.copy_(torch.tensor(at, dtype=torch.int32))
        q.add_(0.25)
        graph.replay()
        assert torch.equal(o, packed_attention(q, k, v, offsets))
        ref, bound = _exact(q, k, v, at, at, True, 0.125)
        _close(o, ref["o"], bound["o"], str(at))


def test_bad_offsets_give_nan(cuda):
    q, k, v, do, _, _ = _inputs([200], [200], 2, 1, 64, torch.bfloat16)
    for at in ([0, 150, 100], [-1, 50, 100], [0, 100, 201]):
        offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = packed_attention(*leaves, offsets)
        assert bool(o.isnan().all())
        assert all(bool(t.isnan().all()) for t in torch.autograd.grad(o, leaves, do))


def test_nothing_to_do(cuda):
    z = lambda n, h: torch.zeros(n, h, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    at = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    assert packed_attention(z(0, 2), z(0, 1), z(0, 1), none).shape == (0, 2, 64)
    assert not packed_attention(z(7, 2), z(7, 1), z(7, 1), none).any()      # no sequence
    q, k = z(7, 2), z(0, 1)
    o = packed_attention(q, k, k, at(0, 3, 7), at(0, 0, 0))
    assert not o.any()
    assert not torch.autograd.grad(o.float().sum(), q)[0].any()
    q, k = z(0, 2), z(5, 1)
    assert not torch.autograd.grad(packed_attention(q, k, k, at(0, 0), at(0, 5)).float().sum(), k)[0].any()


def test_second_derivatives_are_an_error(cuda):
    q, k, v, do, qa, _ = _inputs([40], [40], 2, 2, 64, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = packed_attention(*leaves, torch.tensor(qa, dtype=torch.int32, device="cuda"))
    first = torch.autograd.grad(o, leaves, do.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="packed_attention: its gradient has no gradient"):
        torch.autograd.grad(sum(t.float().sum() for t in first), leaves)


def test_half_precision_gradients_are_refused(cuda):
    q, k, v, _, qa, _ = _inputs([40], [40], 2, 2, 64, torch.float16)
    with pytest.raises(NotImplementedError, match="bf16 only"):
        packed_attention(q.requires_grad_(), k, v, torch.tensor(qa, dtype=torch.int32, device="cuda"))
