"""Gradient norm and clipping (prism_b200.grad_clip) against float64: many tensors of mixed
types, empty and single-element ones, odd sizes and alignments, strides, extreme values and
non-finite ones.

Bounds: the sum is fp64, so the norm is within one fp32 rounding (2^-24, doubled for the final
conversion); the factor adds three more and the output its own type's rounding."""
import pytest
import torch

from prism_b200 import _lib
from prism_b200.grad_clip import clip_grad_norm

pytestmark = pytest.mark.gpu

RND = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def _norm64(grads):
    return float(torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()) if grads else 0.0


def _check(grads, before, outs, norm, max_norm):
    ref = _norm64(before)
    assert norm.dtype == torch.float32 and norm.shape == ()
    assert abs(float(norm) - ref) <= 2.0 ** -23 * ref
    f = min(1.0, max_norm / (ref + 1e-6))
    for b, o in zip(before, outs):
        want = b.double() * f
        bound = (RND[b.dtype] * 1.01 + 6 * 2.0 ** -24) * want.abs() + TINY[b.dtype]
        if f == 1.0:
            assert torch.equal(o, b)
        assert bool(((o.double() - want).abs() <= bound).all())


def _grads(sizes, types, cuda, seed=0, scale=1.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=cuda) * scale).to(types[i % len(types)]) for i, n in enumerate(sizes)]


MIXED = [torch.bfloat16, torch.float32, torch.float16]


@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], [7, 1, 129], [5120] * 9, [32768, 32769, 65535, 65537, 3],
                                   [1_000_003, 17, 4096], list(range(1, 1200)), [2] * 2500])
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9])
def test_mixed_tensors(sizes, max_norm, cuda):
    grads = _grads(sizes, MIXED, cuda)
    before = [g.clone() for g in grads]
    outs = [torch.full_like(g, 7.0) for g in grads]
    norm = clip_grad_norm(grads, max_norm, out=outs)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    _check(grads, before, outs, norm, max_norm)
    again = clip_grad_norm(grads, max_norm)
    assert torch.equal(norm, again) and all(torch.equal(a, b) for a, b in zip(grads, outs))


def test_views_of_one_buffer_at_odd_offsets(cuda):
    """Consecutive odd-sized slices of flat buffers: addresses of every alignment, and nothing
    written between them."""
    sizes = [5, 1, 33, 64, 1027, 8, 2049, 16, 70001]
    for dtype in MIXED:
        flat = _grads([sum(sizes)], [dtype], cuda)[0]
        out = torch.zeros(sum(sizes) + 3, dtype=dtype, device=cuda)
        before, outs = [v.clone() for v in flat.split(sizes)], list(out[3:].split(sizes))
        keep = outs.pop(4)
        grads = list(flat.split(sizes))
        left = [g for i, g in enumerate(grads) if i != 4]
        norm = clip_grad_norm(left, 0.25, out=outs)
        _check(left, [b for i, b in enumerate(before) if i != 4], outs, norm, 0.25)
        assert not bool(out[:3].any()) and not bool(keep.any())


def test_strided_gradients(cuda):
    base = torch.randn(64, 96, generator=torch.Generator().manual_seed(1)).to(cuda)
    wide = torch.randn(50, 200, generator=torch.Generator().manual_seed(2)).to(cuda)
    cube = torch.randn(4, 6, 8, generator=torch.Generator().manual_seed(3)).to(cuda).to(torch.bfloat16)
    grads = [base.t(), wide[:, 10:110], cube.permute(2, 0, 1), torch.randn((), device=cuda)]
    before, edges = [g.clone() for g in grads], wide[:, :10].clone()
    norm = clip_grad_norm(grads, 1.0)
    _check(grads, before, grads, norm, 1.0)
    assert torch.equal(wide[:, :10], edges)
    outs = [torch.empty_like(b, memory_format=torch.contiguous_format) for b in before]
    grads = [b.clone() for b in before[:1]] + [before[1], before[2].transpose(0, 1).contiguous().transpose(0, 1), before[3]]
    norm = clip_grad_norm(grads, 1.0, out=outs)
    _check(grads, before, outs, norm, 1.0)


@pytest.mark.parametrize("scale", [1e-30, 1e-20, 1e18, 1e30])
def test_squares_outside_fp32(scale, cuda):
    """Squares of these values leave fp32's range; the norm does not."""
    for dtype in (torch.float32, torch.bfloat16):
        grads = _grads([1000, 70000, 3], [dtype], cuda, scale=scale)
        before = [g.clone() for g in grads]
        norm = clip_grad_norm(grads, scale)
        ref = _norm64(before)
        assert abs(float(norm) - ref) <= 2.0 ** -23 * ref
        mixed = [grads[0], torch.ones(100, device=cuda), torch.zeros(4096, device=cuda)]
        ref = _norm64(mixed)
        assert abs(float(clip_grad_norm(mixed, float("inf"))) - ref) <= 2.0 ** -23 * ref


def test_non_finite(cuda):
    for bad, at in ((float("nan"), 17), (float("inf"), 40000)):
        grads = _grads([100, 50001], [torch.float32, torch.bfloat16], cuda)
        grads[1][at] = bad
        outs = [torch.empty_like(g) for g in grads]
        norm = clip_grad_norm(grads, 1.0, out=outs)
        ref = torch.nn.utils.get_total_norm([g.float() for g in grads])
        assert bool(norm.isnan()) == bool(ref.isnan()) and (bool(ref.isnan()) or float(norm) == float("inf"))
        f = (1.0 / (norm + 1e-6)).clamp(max=1.0)
        for g, o in zip(grads, outs):
            assert torch.equal((g.float() * f).isnan(), o.isnan())
            assert torch.equal((g.float() * f).nan_to_num(), o.float().nan_to_num())


def test_zero_gradients_and_measuring_only(cuda):
    grads = [torch.zeros(5000, device=cuda), torch.zeros(3, dtype=torch.bfloat16, device=cuda)]
    assert float(clip_grad_norm(grads, 1.0)) == 0.0 and not any(bool(g.any()) for g in grads)
    grads = _grads([4097], [torch.bfloat16], cuda)
    before = grads[0].clone()
    norm = clip_grad_norm(grads, float("inf"))
    _check(grads, [before], grads, norm, float("inf"))
    assert float(clip_grad_norm([], 1.0)) == 0.0
    grads[0][5] = float("inf")
    before = grads[0].clone()
    assert float(clip_grad_norm(grads, float("inf"))) == float("inf") and torch.equal(grads[0], before)


def test_offsets_past_32_bits(cuda):
    g = torch.zeros(2_200_000_007, dtype=torch.bfloat16, device=cuda)
    g[-1], g[0], g[2_150_000_000] = 3.0, 4.0, 12.0
    norm = clip_grad_norm([g], 6.5)
    assert float(norm) == 13.0
    assert (float(g[-1]), float(g[0]), float(g[2_150_000_000])) == (1.5, 2.0, 6.0)


def test_on_a_captured_stream(cuda):
    """The call is capturable: a replay clips what the gradients hold by then."""
    grads = _grads([5000, 33], [torch.float32, torch.bfloat16], cuda)
    clip_grad_norm([g.clone() for g in grads], 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm(grads, 1.0)
    new = _grads([5000, 33], [torch.float32, torch.bfloat16], cuda, seed=9, scale=3.0)
    for g, n in zip(grads, new):
        g.copy_(n)
    graph.replay()
    torch.cuda.synchronize()
    _check(grads, new, grads, norm, 1.0)


def test_refusals(cuda):
    g = torch.ones(4, device=cuda)
    with pytest.raises(ValueError):
        clip_grad_norm([g], -1.0)
    with pytest.raises(ValueError):
        clip_grad_norm([g], float("nan"))
    with pytest.raises(ValueError):
        clip_grad_norm([g], 1.0, out=[])
    with pytest.raises(ValueError):
        clip_grad_norm([g], 1.0, out=[g.to(torch.bfloat16)])
    with pytest.raises(TypeError):
        clip_grad_norm([g.double()], 1.0)
    with pytest.raises(_lib.PrismError):
        clip_grad_norm([g, torch.ones(3)], 1.0)


def test_slices_of_a_flat_buffer_as_outputs(cuda):
    """A 2D gradient into its slice of a flat buffer, row-major whatever the gradient's strides."""
    g = torch.randn(30, 50, generator=torch.Generator().manual_seed(4)).to(cuda)
    for grad in (g, g.t().contiguous().t(), torch.cat((g, g), 1)[:, :50]):
        flat = torch.zeros(1600, device=cuda)
        norm = clip_grad_norm([grad], 0.5, out=[flat[32:1532]])
        _check([grad], [g], [flat[32:1532].view(30, 50)], norm, 0.5)
        assert not bool(flat[:32].any()) and not bool(flat[1532:].any())
    with pytest.raises(ValueError):
        clip_grad_norm([g], 1.0, out=[flat[:1499]])
    with pytest.raises(ValueError):
        clip_grad_norm([g.t()], 1.0, out=[flat[:1499]])
