"""Derivatives of a gradient (create_graph=True) through rotary positions: the rotation is linear, so its
gradient has a gradient."""
import pytest
import torch

from prism_b200.rotary import apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def _turn(x, angle, layout, scale):
    """x [B, S, H, D], angle [S, pairs]: rotated in float64."""
    pairs = angle.shape[-1]
    z = torch.polar(torch.full_like(angle, scale), angle)[None, :, None]
    p = x.unflatten(-1, (pairs, 2)) if layout == "interleaved" else x.unflatten(-1, (2, pairs)).transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(p.contiguous()) * z)
    return y.flatten(-2) if layout == "interleaved" else y.transpose(-1, -2).flatten(-2)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("keys", [False, True])
def test_rotary(layout, keys, cuda):
    """The loss sum a y^3 + q^3 of y = R q has the gradient R'(3 a y^2) + 3 q^2, and that along v the
    gradient R'(6 a y R v) + 6 q v.

    Bound: a rotation is 1e-6 of its pair's |a| + |b| off (angles and products in fp32), three of them
    and a few fp32 products: 1e-5 of the same expression in pair sums of magnitudes."""
    g = torch.Generator(device=cuda).manual_seed(0)
    B, S, H, D, scale = 2, 31, 3, 64, 1.5
    rnd = lambda: torch.randn(B, S, H, D, generator=g, device=cuda)
    q, a, v = rnd().requires_grad_(), rnd(), rnd()
    k = rnd().requires_grad_() if keys else None
    freqs, _ = rotary_frequencies(D, device=cuda)
    pos = torch.arange(S, device=cuda) + 1000
    y, ky = apply_rotary(q, k, pos, freqs, layout=layout, scale=scale)
    loss = (a * y ** 3).sum() + (q ** 3).sum() + ((ky ** 2).sum() if keys else 0)
    wanted = (q, k) if keys else (q,)
    grads = torch.autograd.grad(loss, wanted, create_graph=True)
    second = torch.autograd.grad((grads[0] * v).sum(), q, retain_graph=True)[0]
    angle = pos.double()[:, None] * freqs
    turn = lambda x, sign=1.0: _turn(x.double(), sign * angle, layout, scale)
    with torch.no_grad():
        q64, a64, v64 = q.double(), a.double(), v.double()
        y64 = turn(q64)
        first = turn(3 * a64 * y64 ** 2, -1.0) + 3 * q64 ** 2
        ref = turn(6 * a64 * y64 * turn(v64), -1.0) + 6 * q64 * v64

        def sums(x):   # |a| + |b| of each pair, at both its places
            x = x.abs()
            if layout == "interleaved":
                return scale * x.unflatten(-1, (D // 2, 2)).sum(-1, keepdim=True).expand(B, S, H, D // 2, 2).flatten(-2)
            return scale * (x + x.roll(D // 2, -1))
        size1 = sums(3 * a64.abs() * sums(q64) ** 2) + 3 * q64 ** 2
        size2 = sums(6 * a64.abs() * sums(q64) * sums(v64)) + (6 * q64 * v64).abs()
        assert bool(((grads[0].double() - first).abs() <= 1e-5 * size1).all())
        assert bool(((second.double() - ref).abs() <= 1e-5 * size2).all())
    if keys:   # sum (R k)^2 = scale^2 sum k^2: gradient 2 scale^2 k, along v 2 scale^2 v
        second = torch.autograd.grad((grads[1] * v).sum(), k)[0]
        with torch.no_grad():
            assert bool(((second.double() - 2 * scale ** 2 * v64).abs() <= 1e-5 * 2 * sums(sums(v64))).all())


def test_only_one_rotated_tensor(cuda):
    """The gradient of k's rotation alone has its gradient, too."""
    g = torch.Generator(device=cuda).manual_seed(1)
    q, k, v = (torch.randn(1, 9, 2, 32, generator=g, device=cuda) for _ in range(3))
    q.requires_grad_(), k.requires_grad_()
    freqs, _ = rotary_frequencies(32, device=cuda)
    ky = apply_rotary(q, k, torch.arange(9, device=cuda), freqs)[1]
    grad = torch.autograd.grad((ky ** 2).sum(), k, create_graph=True)[0]
    second = torch.autograd.grad((grad * v).sum(), k)[0]
    size = v.abs().unflatten(-1, (16, 2)).sum(-1, keepdim=True).expand(1, 9, 2, 16, 2).flatten(-2)
    assert bool(((second - 2 * v).abs() <= 1e-5 * 4 * size).all())
