"""Clipping moves the version counter of what it writes, so that autograd refuses a graph that saved
the old values."""
import pytest
import torch

from prism_b200 import clip_grad_norm

pytestmark = pytest.mark.gpu


def test_in_place(cuda):
    p = torch.ones(500, device=cuda, requires_grad=True)
    for g in (torch.full((500,), 3.0, device=cuda), torch.full((500, 2), 3.0, device=cuda)[:, 0]):
        loss = (p * g).sum()            # saves g for p's gradient
        before = g._version
        clip_grad_norm([g], 1.0)
        assert g._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss, p)


def test_outputs(cuda):
    g, flat = torch.full((500,), 3.0, device=cuda), torch.zeros(600, device=cuda)
    before = g._version, flat._version
    clip_grad_norm([g], 1.0, out=[flat[50:550]])
    assert g._version == before[0] and flat._version > before[1]


def test_measuring_alone_writes_nothing(cuda):
    for g in (torch.full((500,), 3.0, device=cuda), torch.full((500, 2), 3.0, device=cuda)[:, 0]):
        before = g._version
        clip_grad_norm([g], float("inf"))
        assert g._version == before


def test_inference_tensors(cuda):
    with torch.inference_mode():
        g = torch.full((500,), 3.0, device=cuda)
        clip_grad_norm([g], 1.0)
    clip_grad_norm([g], 0.5)
    assert abs(float(g.norm()) - 0.5) <= 1e-5
