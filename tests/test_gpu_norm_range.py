"""RMS norm of finite rows whose squares leave fp32: forward, 8-bit rows and gradients against
float64, next to rows of ordinary size.

Bounds: those of the ordinary range -- a = (cols / 32 + 64) 2^-24 bounds the relative error of an
fp32 row sum; half a unit in the last place for the output; half the least subnormal where the gradient
gets that small (it is of order 1 / |h|), and 2^-149 for each of some eight products on its way."""
import pytest
import torch

from prism_b200.norm import add_rms_norm, add_rms_norm_fp8

pytestmark = pytest.mark.gpu

RND = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float32)}
TINY = {torch.bfloat16: 2.0 ** -134 + 8 * 2.0 ** -149, torch.float32: 9 * 2.0 ** -149}
EPS = 1e-6


def _inputs(cols, dtype, size, cuda):
    """37 rows, of which every third has elements up to `size` and the last one is 2^-20 of that."""
    g = torch.Generator(device=cuda).manual_seed(cols)
    x = torch.rand(37, cols, generator=g, device=cuda) * 2 - 1
    x[::3] *= size
    x[-1] = (torch.rand(cols, generator=g, device=cuda) * 2 - 1) * (size * 2.0 ** -20)
    r = torch.randn(37, cols, generator=g, device=cuda)
    w = 1 + 0.3 * torch.randn(cols, generator=g, device=cuda)
    gy = torch.randn(37, cols, generator=g, device=cuda)
    return x.to(dtype), r.to(dtype), w, gy.to(dtype)


def _a(cols):
    return (cols / 32 + 64) * 2.0 ** -24


@pytest.mark.parametrize("dtype", list(RND))
@pytest.mark.parametrize("cols", [8, 96, 193, 1535, 1536, 5120, 20011])
@pytest.mark.parametrize("size", [1e16, 1e22, 1e25, 3e38])
@pytest.mark.parametrize("residual", [False, True])
def test_against_float64(cols, dtype, size, residual, cuda):
    x, r, w, gy = _inputs(cols, dtype, size, cuda)
    x.requires_grad_(), w.requires_grad_()
    r = r if residual else None
    y, h = add_rms_norm(x, r, w, EPS)
    dx, dw = torch.autograd.grad(y, (x, w), gy)
    with torch.no_grad():
        h64 = h.double()
        assert residual or torch.equal(h, x)
        assert not residual or torch.equal(h64, (x.double() + r.double()).to(dtype).double())
        u = 1 / (h64.square().mean(-1, keepdim=True) + EPS).sqrt()
        y64 = h64 * u * w.double()
        assert bool(((y.double() - y64).abs() <= (RND[dtype] * 1.01 + _a(cols)) * y64.abs() + TINY[dtype]).all())

        y8, s, h8 = add_rms_norm_fp8(x, r, w, EPS)
        s64 = y64.abs().amax(-1, keepdim=True) / 448
        assert torch.equal(h8, h)
        assert bool(((s.double()[:, None] - s64).abs() <= (_a(cols) + 2.0 ** -21) * s64).all())
        v = y64 / s64
        assert bool(((y8.float().double() - v).abs() <= 2.0 ** -4 * v.abs() + 2.0 ** -10 + 2 * _a(cols) * v.abs()).all())

        g, along = gy.double() * w.double(), gy.double() * w.double() * h64 * u
        ref = g * u - h64 * u * u / cols * along.sum(-1, keepdim=True)
        each = (g * u).abs() + (h64 * u * u).abs() / cols * along.abs().sum(-1, keepdim=True)
        off = (dx.double() - ref).abs() / (RND[dtype] * 1.01 * ref.abs() + 4 * _a(cols) * each + TINY[dtype])
        assert float(off.max()) <= 1, (float(off.max()), int(off.amax(-1).argmax()))
        parts = gy.double() * h64 * u
        assert bool(((dw.double() - parts.sum(0)).abs() <= ((37 + 64) * 2.0 ** -24 + _a(cols)) * parts.abs().sum(0)).all())


def test_infinities_among_large_values(cuda):
    """A row with an infinity still has scale NaN, and NaN at the infinity; its neighbours are theirs."""
    x, _, w, _ = _inputs(1536, torch.float32, 1e25, cuda)
    clean, clean8 = add_rms_norm(x, None, w, EPS)[0], add_rms_norm_fp8(x, None, w, EPS)
    x[3, 7], x[6, 9] = float("inf"), float("nan")
    y, (y8, s, _) = add_rms_norm(x, None, w, EPS)[0], add_rms_norm_fp8(x, None, w, EPS)
    rest = torch.tensor([i for i in range(37) if i not in (3, 6)], device=cuda)
    assert bool(s[[3, 6]].isnan().all()) and bool(y[3, 7].isnan()) and bool(y[6].isnan().all())
    assert torch.equal(y[rest], clean[rest]) and torch.equal(s[rest], clean8[1][rest])
    assert torch.equal(y8[rest].float(), clean8[0][rest].float())
