"""The operators around the attention on a stream of their own, behind a queue of products that keeps
their inputs from being there yet: a launch on any other stream would read zeros."""
import pytest
import torch

from prism_b200 import (add_rms_norm, add_rms_norm_fp8, apply_rotary, clip_grad_norm, linear_fp8, quantize_rows_fp8,
                        rotary_frequencies)

pytestmark = pytest.mark.gpu


def _norm(x, r):
    return add_rms_norm(x, r)


def _norm_8bit(x, r):
    y8, s, h = add_rms_norm_fp8(x, r)
    return y8.float(), s, h


def _norm_backward(x, r):
    x.requires_grad_()
    w = torch.ones(x.shape[-1], device=x.device, requires_grad=True)
    out = torch.autograd.grad(add_rms_norm(x, r, w), (x, w), (r, x.detach()))
    x.requires_grad_(False)
    return out


def _rotary(x, r):
    q, k = x.view(-1, 8, 64), r.view(-1, 8, 64)
    freqs, _ = rotary_frequencies(64, device=x.device)
    return apply_rotary(q, k, torch.arange(len(q), device=x.device), freqs)


def _rotary_backward(x, r):
    q = x.view(-1, 8, 64).detach().requires_grad_()
    freqs, _ = rotary_frequencies(64, device=x.device)
    y = apply_rotary(q, None, torch.arange(len(q), device=x.device), freqs)[0]
    return torch.autograd.grad(y, q, r.view(-1, 8, 64))


def _projection(x, r):
    return linear_fp8(*quantize_rows_fp8(x), *quantize_rows_fp8(r[:512])),


def _clip(x, r):
    out = [torch.empty_like(x), torch.empty_like(r)]
    return clip_grad_norm([x, r], 1.0, out=out), *out


@pytest.mark.parametrize("op", [_norm, _norm_8bit, _norm_backward, _rotary, _rotary_backward, _projection, _clip])
def test_on_another_stream(op, cuda):
    g = torch.Generator(device=cuda).manual_seed(0)
    x, r = (torch.randn(1000, 512, generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
    want = op(x, r)
    late = [torch.zeros_like(t) for t in (x, r)]
    busy = torch.randn(8192, 8192, generator=g, device=cuda).to(torch.bfloat16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):   # some 14 ms
            busy @ busy
        for a, b in zip(late, (x, r)):
            a.copy_(b)
        got = op(*late)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
