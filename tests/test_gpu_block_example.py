"""The operators together as a block uses them (examples/transformer_block.py): a training step's
gradients against the same block in float64 torch, a falling loss under clipping, and the 8-bit
inference form against the 16-bit one."""
import os
import sys

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
from transformer_block import Block, data, train  # noqa: E402


def _reference(block, params, x):
    """The block with every key attended, in float64."""
    S, dim = x.shape
    heads, D = block.heads, dim // block.heads
    norm = lambda h, w: h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
    axis = torch.repeat_interleave(torch.arange(3), torch.tensor(block.sections)).to(x.device)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       block.positions.double()[:, axis] * block.freqs)[:, None]
    rotate = lambda t: torch.view_as_real(torch.view_as_complex(t.unflatten(-1, (D // 2, 2)).contiguous()) * turn).flatten(-2)
    q, k, v = (norm(x, params["norm_1"]) @ params["qkv"].t()).view(S, 3, heads, D).unbind(1)
    q, k, v = rotate(q).transpose(0, 1), rotate(k).transpose(0, 1), v.transpose(0, 1)
    o = ((q @ k.transpose(1, 2) * D ** -0.5).softmax(-1) @ v).transpose(0, 1).reshape(S, dim)
    h = x + o @ params["o"].t()
    return F.gelu(norm(h, params["norm_2"]) @ params["up"].t()) @ params["down"].t() + h


def test_gradients_of_the_whole_block(cuda):
    """bf16 roundings (2^-8 each) of some ten intermediate tensors: 3e-2 relative L2 for every
    gradient."""
    block = Block((4, 8, 8), sparsity=0.0)
    x, target = data(block.grid, 256)
    p64 = {n: p.detach().double().requires_grad_() for n, p in block.params.items()}
    ref = torch.autograd.grad(F.mse_loss(_reference(block, p64, x.double()), target.double()), list(p64.values()))
    params = list(block.params.values())
    for p in params:
        p.requires_grad_()
    delta, h = block.forward(torch.zeros_like(x), x)
    got = torch.autograd.grad(F.mse_loss((delta + h).float(), target), params)
    for name, a, b in zip(p64, got, ref):
        rel = float((a.double() - b).norm() / b.norm())
        assert rel <= 3e-2, (name, rel)


@pytest.mark.parametrize("max_norm", [0.05, 10.0])
def test_training(max_norm, cuda):
    """Small steps of gradient descent lower the loss by what the first order says: the step's
    length lr min(|g|, max_norm) along g times |g|.  Half and one and a half of it are allowed for
    the curvature and the bf16 noise of the loss."""
    block = Block((4, 8, 8), sparsity=0.0)
    x, target = data(block.grid, 256)
    lr = 0.2
    log = train(block, x, target, 9, lr=lr, max_norm=max_norm)
    expected = sum(lr * min(n, max_norm) * n for _, n in log[:-1])
    assert 0.5 * expected <= log[0][0] - log[-1][0] <= 1.5 * expected


def test_8bit_inference(cuda):
    """8-bit rows are 2^-4 / sqrt(3) off at most in relative L2 (3.6e-2, uniform errors of half a
    unit), on both sides of each of the four products in line: 0.15 for the block's output."""
    block = Block((4, 8, 8), sparsity=0.0)
    x, target = data(block.grid, 256)
    with torch.no_grad():
        ref, h = block.forward(torch.zeros_like(x), x)
    got, h8 = block.forward_8bit(torch.zeros_like(x), x, block.quantized())
    assert float((got.double() - ref.double()).norm() / ref.double().norm()) <= 0.15
    assert float((h8.double() - h.double()).norm() / h.double().norm()) <= 0.15
