"""One video transformer block on the package's operators: training steps, and the 8-bit
inference form of the same weights.

    python examples/transformer_block.py [--steps N]

A block here is attention and a feed-forward layer on a residual stream:

    y, h = add_rms_norm(delta, h, w)           residual + norm, one pass
    q, k, v = linear(y, ...)                   tensor-core projections
    q, k = apply_rotary(q, k, positions, ...)  frame / row / column positions
    o = run_bsa_uniform(q, k, v, grid, ...)    block-sparse attention
    delta = linear(o, ...)                     and likewise the feed-forward layer

The training step ends with ``clip_grad_norm`` over every gradient, into the flat buffer that the
update reads.  In inference the two norms write 8-bit rows, which ``linear_fp8`` multiplies by
8-bit weights.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from prism_b200 import (  # noqa: E402
    add_rms_norm, add_rms_norm_fp8, apply_rotary, clip_grad_norm, linear_fp8, quantize_rows_fp8,
                        rotary_frequencies, run_bsa_uniform)
from prism_b200.linear import linear  # noqa: E402

CHUNK = (4, 4, 4)


class Block:
    def __init__(self, grid, heads: int = 4, head_dim: int = 64, ffn: int = 512, sparsity: float = 0.5, seed: int = 0,
                 device="cuda"):
        dim = heads * head_dim
        g = torch.Generator(device=device).manual_seed(seed)
        weight = lambda n, k: torch.randn(n, k, generator=g, device=device) * k ** -0.5
        self.grid, self.heads, self.sparsity = grid, heads, sparsity
        self.params = {"norm_1": torch.ones(dim, device=device), "norm_2": torch.ones(dim, device=device),
                       "qkv": weight(3 * dim, dim), "o": weight(dim, dim), "up": weight(ffn, dim),
                       "down": weight(dim, ffn)}
        # the pairs of a head follow the frame, the row and the column, as the video layer splits them
        third = head_dim // 3 // 2 * 2
        dims = (head_dim - 2 * third, third, third)
        self.freqs = torch.cat([rotary_frequencies(d, device=device)[0] for d in dims])
        self.sections = tuple(d // 2 for d in dims)
        T, H, W = grid
        at = torch.arange(T * H * W, device=device)
        self.positions = torch.stack([at // (H * W), at // W % H, at % W], -1)

    def _weights(self):
        """fp32 parameters as the layers read them: matrices in bf16."""
        return {n: p.to(torch.bfloat16) if p.dim() == 2 else p for n, p in self.params.items()}

    def _attention(self, qkv):
        S = qkv.shape[0]
        q, k, v = qkv.view(S, 3, self.heads, -1).unbind(1)
        q, k = apply_rotary(q, k, self.positions, self.freqs, sections=self.sections)
        o = run_bsa_uniform(q[None], k[None], v[None], self.grid, layout="bshd", sparsity=self.sparsity,
                            cdf_threshold=None, chunk_3d_shape_q=CHUNK, chunk_3d_shape_k=CHUNK)
        return o.reshape(S, -1)

    def forward(self, delta, h):
        """(the feed-forward layer's output, the residual stream): the next block's inputs."""
        p = self._weights()
        y, h = add_rms_norm(delta, h, p["norm_1"])
        delta = linear(self._attention(linear(y, p["qkv"])), p["o"])
        y, h = add_rms_norm(delta, h, p["norm_2"])
        return linear(F.gelu(linear(y, p["up"])), p["down"]), h

    def quantized(self):
        """The weights' 8-bit rows and scales, laid out once."""
        return {n: quantize_rows_fp8(self.params[n].detach()) for n in ("qkv", "o", "up", "down")}

    @torch.no_grad()
    def forward_8bit(self, delta, h, weights):
        p = self.params
        y8, scale, h = add_rms_norm_fp8(delta, h, p["norm_1"])
        o = self._attention(linear_fp8(y8, scale, *weights["qkv"]))
        delta = linear_fp8(*quantize_rows_fp8(o), *weights["o"])
        y8, scale, h = add_rms_norm_fp8(delta, h, p["norm_2"])
        return linear_fp8(*quantize_rows_fp8(F.gelu(linear_fp8(y8, scale, *weights["up"]))), *weights["down"]), h


def train(block: Block, x, target, steps: int, lr: float = 0.3, max_norm: float = 1.0):
    """Plain gradient descent on the mean square error: [(loss, gradient norm)] of the steps."""
    params = list(block.params.values())
    for p in params:
        p.requires_grad_()
    sizes = [p.numel() for p in params]
    clipped = torch.zeros(sum(sizes), device=x.device).split(sizes)   # the optimizer's flat buffer
    log = []
    for _ in range(steps):
        delta, h = block.forward(torch.zeros_like(x), x)
        loss = F.mse_loss((delta + h).float(), target)
        grads = torch.autograd.grad(loss, params)
        norm = clip_grad_norm(grads, max_norm, out=clipped)
        with torch.no_grad():
            for p, g in zip(params, clipped):
                p.sub_(lr * g.view_as(p))
        log.append((loss.detach(), norm))
    return [(float(a), float(b)) for a, b in log]


def data(grid, dim: int, seed: int = 1, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    S = grid[0] * grid[1] * grid[2]
    x = torch.randn(S, dim, generator=g, device=device).to(torch.bfloat16)
    return x, x.float().roll(1, 0) * 0.5 + x.float()


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    block = Block(grid=(4, 8, 8))
    x, target = data(block.grid, 256)
    for i, (loss, norm) in enumerate(train(block, x, target, a.steps)):
        print(f"step {i:3d}  loss {loss:.4f}  gradient norm {norm:.3f}")
    with torch.no_grad():
        ref, _ = block.forward(torch.zeros_like(x), x)
    got, _ = block.forward_8bit(torch.zeros_like(x), x, block.quantized())
    print(f"8-bit block output against bf16: relative L2 {float((got.float() - ref.float()).norm() / ref.float().norm()):.4f}")


if __name__ == "__main__":
    main()
