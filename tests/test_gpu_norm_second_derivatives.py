"""Derivatives of a gradient (create_graph=True) through the RMS norm, whose gradient has none: asking
for it is an error, also where the loss reaches the inputs by another path."""
import pytest
import torch

from prism_b200.norm import add_rms_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("residual", [False, True])
def test_norm_refuses(residual, cuda):
    g = torch.Generator(device=cuda).manual_seed(2)
    x, r = (torch.randn(7, 96, generator=g, device=cuda).requires_grad_() for _ in range(2))
    w = torch.ones(96, device=cuda).requires_grad_()
    r = r if residual else None
    wanted = [t for t in (x, r, w) if t is not None]
    # h is x itself without a residual: another path to the inputs
    loss = lambda y, h: (y ** 3).sum() + (h ** 3).sum() + (w ** 3).sum()
    plain = torch.autograd.grad(loss(*add_rms_norm(x, r, w)), wanted)
    grads = torch.autograd.grad(loss(*add_rms_norm(x, r, w)), wanted, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, grads))   # the first derivatives stay as they are
    for grad in grads:
        with pytest.raises(RuntimeError, match="add_rms_norm"):
            torch.autograd.grad(grad.square().sum(), wanted, retain_graph=True, allow_unused=True)


def test_the_residual_stream_alone(cuda):
    """h = x + r is linear: where y has no part in the loss its gradient has a gradient."""
    g = torch.Generator(device=cuda).manual_seed(3)
    x, r = (torch.randn(5, 64, generator=g, device=cuda).requires_grad_() for _ in range(2))
    h = add_rms_norm(x, r)[1]
    grad = torch.autograd.grad((h ** 3).sum(), x, create_graph=True)[0]
    second = torch.autograd.grad(grad.sum(), r)[0]
    assert torch.equal(second, 6 * h.detach())
