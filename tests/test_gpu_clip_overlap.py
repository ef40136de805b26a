"""Clipping lists whose entries share memory: what is given twice counts twice and is scaled once; what
overlaps otherwise is refused before anything is written.  Bounds as for other lists: the norm within 2^-23, an
output within its type's rounding and six fp32 ones."""
import random

import pytest
import torch

from prism_b200 import _lib, add_rms_norm, clip_grad_norm

pytestmark = pytest.mark.gpu


def _close(got, want):
    eps = torch.finfo(got.dtype).eps / 2 * 1.01 + 6 * 2.0 ** -24
    return bool(((got.double() - want).abs() <= eps * want.abs()).all())


def test_gradients_of_the_norms_two_inputs(cuda):
    """dL/dx and dL/dr of h = x + r are one tensor."""
    g = torch.Generator(device=cuda).manual_seed(0)
    x, r, gy, gh = (torch.randn(300, 1024, generator=g, device=cuda).to(torch.bfloat16) for _ in range(4))
    x.requires_grad_(), r.requires_grad_()
    w = torch.ones(1024, device=cuda, requires_grad=True)
    for _ in range(20):
        grads = torch.autograd.grad(add_rms_norm(x, r, w), (x, r, w), (gy, gh))
        assert grads[0].data_ptr() == grads[1].data_ptr()
        before = [t.double().clone() for t in grads]
        norm = clip_grad_norm(grads, 0.5)
        ref = float(sum(b.square().sum() for b in before).sqrt())
        assert abs(float(norm) - ref) <= 2.0 ** -23 * ref
        assert all(_close(t, b * (0.5 / (ref + 1e-6))) for t, b in zip(grads, before))


@pytest.mark.parametrize("count", [3, 500])
def test_many_repeated_in_any_order(count, cuda):
    g = torch.Generator(device=cuda).manual_seed(1)
    flat = torch.randn(count * 1000, generator=g, device=cuda)
    parts = list(flat.split(1000))
    rng = random.Random(2)
    grads = [p.view(8, 125) if i % 3 == 0 else p for i, p in enumerate(parts)] + [rng.choice(parts) for _ in range(count)]
    grads += [parts[0].view(8, 125).t(), flat[:0]]
    rng.shuffle(grads)
    before = [t.double().clone() for t in grads]
    norm = clip_grad_norm(grads, 2.0)
    ref = float(torch.cat([b.flatten() for b in before]).norm())
    assert abs(float(norm) - ref) <= 2.0 ** -23 * ref
    assert all(_close(t, b * (2.0 / (ref + 1e-6))) for t, b in zip(grads, before))
    # apart from each other: the same list into outputs of its own
    outs = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in grads]
    now = [t.double().clone() for t in grads]
    norm = clip_grad_norm(grads, 1.0, out=outs)
    ref = float(torch.cat([b.flatten() for b in now]).norm())
    assert all(_close(o, b * (1.0 / (ref + 1e-6))) for o, b in zip(outs, now))
    assert all(torch.equal(t.double(), b) for t, b in zip(grads, now))


def test_strided_views_that_overlap(cuda):
    """Views with gaps go through copies: each counts, and what two of them share is scaled once."""
    wide = torch.randn(50, 200, generator=torch.Generator().manual_seed(3)).to(cuda)
    grads = [wide[:, 10:110], wide[:, 50:150]]
    before, whole = [t.double().clone() for t in grads], wide.double().clone()
    norm = clip_grad_norm(grads, 1.0)
    ref = float(torch.cat([b.flatten() for b in before]).norm())
    assert abs(float(norm) - ref) <= 2.0 ** -23 * ref
    assert all(_close(t, b / (ref + 1e-6)) for t, b in zip(grads, before))
    assert torch.equal(wide[:, :10].double(), whole[:, :10]) and torch.equal(wide[:, 150:].double(), whole[:, 150:])


def test_refusals_write_nothing(cuda):
    flat = torch.randn(10000, generator=torch.Generator().manual_seed(4)).to(cuda)
    before = flat.clone()
    a, b = flat[:6000], flat[4000:]
    for grads, outs in (([a, b], None), ([a[:100], b], [flat[50:150], b]), ([a[:100], a[100:200]], [flat[300:400]] * 2),
                        ([a], [flat[1:6001]])):
        with pytest.raises(_lib.PrismError, match="overlap"):
            clip_grad_norm(grads, 1.0, out=outs)
    torch.cuda.synchronize()
    assert torch.equal(flat, before)
    # nothing is written where the norm is only measured
    ref = float(torch.cat([a, b]).double().norm())
    assert abs(float(clip_grad_norm([a, b], float("inf"))) - ref) <= 2.0 ** -23 * ref
    assert torch.equal(flat, before)
