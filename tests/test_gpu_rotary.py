"""Rotary positions (prism_b200.rotary) against complex multiplication in float64: layouts, part
of the head, sections over position axes, long positions, strides, shared key heads, and the
gradient.

Bound: the angle is reduced in fp64 and rounded to fp32 in turns (at most 2^-26 turns off, 1e-7
rad), cos and sin add two units in the last place and the products three roundings: below
1e-6 scale (|a| + |b|) for a pair (a, b), plus the output's rounding."""
import pytest
import torch

from prism_b200 import _lib
from prism_b200.rotary import apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu

RND = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def _reference(x, pos, freqs, layout, sections, scale, conjugate=False):
    """x [B, S, H, D]; pos [B, S, axes] -> (rotated, |a| + |b| per rotated column) in float64."""
    pairs = freqs.shape[0]
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(x.device)
    angle = pos.double()[..., axis] * freqs
    turn = torch.polar(torch.full_like(angle, scale), -angle if conjugate else angle)[:, :, None]
    x = x.double()
    rot = x[..., :2 * pairs]
    pair = rot.unflatten(-1, (pairs, 2)) if layout == "interleaved" else rot.unflatten(-1, (2, pairs)).transpose(-1, -2)
    y = torch.view_as_real(torch.complex(pair[..., 0], pair[..., 1]) * turn)
    size = (pair.abs().sum(-1, keepdim=True) * scale).expand_as(pair)
    back = (lambda t: t.flatten(-2)) if layout == "interleaved" else (lambda t: t.transpose(-1, -2).flatten(-2))
    return torch.cat((back(y), x[..., 2 * pairs:]), -1), torch.cat((back(size), torch.zeros_like(x[..., 2 * pairs:])), -1)


def _check(got, x, *spec, what="", **kw):
    ref, size = _reference(x, *spec, **kw)
    bound = RND[got.dtype] * ref.abs() * 1.01 + 1e-6 * size + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    assert bool(((got.double() - ref).abs() <= bound).all()), \
        (what, float(((got.double() - ref).abs() / bound.clamp_min(1e-300)).max()))
    rot = 2 * spec[1].shape[0]
    assert torch.equal(got[..., rot:], x[..., rot:])


CASES = [  # B, S, Hq, Hk, D, rot, first position
    (1, 1, 1, 1, 2, 2, 0), (2, 1, 8, 2, 128, 128, 1_000_003), (1, 77, 5, 1, 80, 60, 3), (3, 65, 4, 4, 64, 64, 9),
    (2, 33, 3, 3, 96, 24, 131_000), (1, 130, 2, 1, 256, 192, 0), (1, 50, 7, 7, 36, 34, 5), (1, 9, 2, 2, 7, 6, 1),
    (1, 40, 40, 40, 128, 128, 0), (2, 0, 2, 2, 64, 64, 0), (4, 300, 1, 1, 32, 16, 2_000_000_000),
]


@pytest.mark.parametrize("B,S,hq,hk,D,rot,first", CASES)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", list(RND))
def test_forward_and_gradient(B, S, hq, hk, D, rot, first, layout, dtype, cuda):
    g = torch.Generator(device=cuda).manual_seed(B + S + D)
    rnd = lambda h: torch.randn(B, S, h, D, generator=g, device=cuda).to(dtype)
    q, k, gq, gk = rnd(hq).requires_grad_(), rnd(hk).requires_grad_(), rnd(hq), rnd(hk)
    freqs, _ = rotary_frequencies(rot, device=cuda)
    pos = first + torch.arange(S, device=cuda) + 11 * torch.arange(B, device=cuda)[:, None]
    scale = 1.25
    qo, ko = apply_rotary(q, k, pos, freqs, layout=layout, scale=scale)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk))
    spec = (pos[..., None], freqs, layout, (rot // 2,), scale)
    _check(qo.detach(), q.detach(), *spec, what="q")
    _check(ko.detach(), k.detach(), *spec, what="k")
    _check(dq, gq, *spec, conjugate=True, what="dq")
    _check(dk, gk, *spec, conjugate=True, what="dk")


@pytest.mark.parametrize("sections", [(22, 21, 21), (64, 0, 0), (0, 32, 32), (1, 62, 1), (40, 24), (64,)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_sections(sections, layout, cuda):
    """Frame / row / column positions; (22, 21, 21) with interleaved pairs is the video layer's split."""
    g = torch.Generator(device=cuda).manual_seed(1)
    q = torch.randn(1, 60, 3, 128, generator=g, device=cuda).to(torch.bfloat16)
    axes = len(sections)
    pos = torch.randint(0, 1024, (1, 60, axes), generator=g, device=cuda)
    freqs, _ = rotary_frequencies(128, device=cuda)
    out, none = apply_rotary(q, None, pos, freqs, layout=layout, sections=sections)
    assert none is None
    _check(out, q, pos, freqs, layout, sections, 1.0)
    # positions without the batch, 32-bit, and with the axes in another memory order
    other = pos[0].to(torch.int32).t().contiguous().t()
    assert torch.equal(apply_rotary(q, None, other, freqs, layout=layout, sections=sections)[0], out)


def test_the_layers_table_form(cuda):
    """With its frequencies and sections, the operator rotates as the layer's stored table does."""
    from prism_b200.producer import rope_table
    grid, D = (3, 5, 7), 128
    table = rope_table(grid, D, device=cuda)
    third = D // 3
    dims = (D - 2 * third, third, third)
    freqs = torch.cat([rotary_frequencies(d, device=cuda)[0] for d in dims])
    at = torch.arange(105, device=cuda)
    pos = torch.stack([at // 35, at // 7 % 5, at % 7], -1)
    q = torch.randn(105, 4, D, generator=torch.Generator().manual_seed(0)).to(cuda)
    got, _ = apply_rotary(q, None, pos, freqs, sections=[d // 2 for d in dims])
    z = torch.view_as_complex(q.double().unflatten(-1, (D // 2, 2))) * torch.view_as_complex(table)[:, None]
    assert float((got.double() - torch.view_as_real(z).flatten(-2)).abs().max()) <= 1e-5


def test_strides(cuda):
    """Slices of a fused projection, head-major tensors, unaligned heads and odd offsets."""
    g = torch.Generator(device=cuda).manual_seed(2)
    freqs, _ = rotary_frequencies(64, device=cuda)
    pos = torch.arange(50, device=cuda, dtype=torch.int32) * 3
    qkv = torch.randn(2, 50, 12, 64, generator=g, device=cuda).to(torch.bfloat16)
    spec = (pos.expand(2, 50)[..., None], freqs, "half", (32,), 1.0)
    q, k = apply_rotary(qkv[:, :, :8], qkv[:, :, 8:10], pos, freqs, layout="half")
    _check(q, qkv[:, :, :8], *spec)
    _check(k, qkv[:, :, 8:10], *spec)
    head_major = qkv.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(apply_rotary(head_major, None, pos, freqs, layout="half")[0][:, :, :8], q)
    wide = torch.randn(2, 50, 12, 67, generator=g, device=cuda).to(torch.bfloat16)
    odd = wide[..., 1:65]
    _check(apply_rotary(odd, None, pos, freqs, layout="half")[0], odd, *spec)
    flipped = qkv.transpose(-1, -2).contiguous().transpose(-1, -2)   # columns not contiguous
    assert torch.equal(apply_rotary(flipped, None, pos, freqs, layout="half")[0][:, :, :8], q)
    one = qkv[:, :1].expand(2, 50, 12, 64)                            # zero token stride
    _check(apply_rotary(one, None, pos, freqs, layout="half")[0], one, *spec)
    q3, k3 = apply_rotary(qkv[0, :, :8], qkv[0, :, 8:10], pos, freqs, layout="half")
    assert torch.equal(q3, q[0]) and torch.equal(k3, k[0])


def test_only_one_gradient(cuda):
    freqs, _ = rotary_frequencies(64, device=cuda)
    q = torch.randn(1, 9, 2, 64, device=cuda, requires_grad=True)
    k = torch.randn(1, 9, 1, 64, device=cuda, requires_grad=True)
    pos = torch.arange(9, device=cuda)
    spec = (pos[None, :, None], freqs, "interleaved", (32,), 1.0)
    for wrt, i in ((q, 0), (k, 1)):
        out = apply_rotary(q, k, pos, freqs)[i]
        grad = torch.autograd.grad(out, wrt, torch.ones_like(out))[0]
        _check(grad, torch.ones_like(wrt), *spec, conjugate=True)
    out = apply_rotary(q, k.detach(), pos, freqs)
    assert torch.autograd.grad(out[0].sum(), q)[0].shape == q.shape


def test_gradient_against_differences(cuda):
    """The operator is linear, so a difference of any step is its derivative: <y(q + v) - y(q), a>
    = <grad, v> up to fp32 roundings (2^-23 per element, n = 6,400 elements)."""
    g = torch.Generator(device=cuda).manual_seed(3)
    freqs, _ = rotary_frequencies(48, device=cuda)
    q, v, a = (torch.randn(2, 10, 5, 64, generator=g, device=cuda) for _ in range(3))
    pos = torch.arange(10, device=cuda) + 100_000
    q.requires_grad_()
    y = apply_rotary(q, None, pos, freqs, layout="half", scale=0.7)[0]
    grad = torch.autograd.grad(y, q, a)[0]
    with torch.no_grad():
        moved = apply_rotary(q + v, None, pos, freqs, layout="half", scale=0.7)[0]
        diff = float(((moved.double() - y.double()) * a.double()).sum())
        got = float((grad.double() * v.double()).sum())
    assert abs(diff - got) <= 8 * 2.0 ** -23 * q.numel() ** 0.5 * 8


def test_offsets_past_32_bits(cuda):
    S, H, D = 420_001, 40, 128           # 2.15e9 elements
    q = torch.ones(S, H, D, dtype=torch.bfloat16, device=cuda)
    freqs, _ = rotary_frequencies(D, device=cuda)
    pos = torch.arange(S, device=cuda)
    out, _ = apply_rotary(q, None, pos, freqs)
    _check(out[None, -2:], q[None, -2:], pos[None, -2:, None], freqs, "interleaved", (64,), 1.0)


def test_refusals(cuda):
    q = torch.zeros(4, 2, 64, device=cuda)
    pos = torch.arange(4, device=cuda)
    freqs, _ = rotary_frequencies(64, device=cuda)
    with pytest.raises(ValueError):
        apply_rotary(q, None, pos, freqs, layout="columns")
    with pytest.raises(ValueError):
        apply_rotary(q, None, pos[:3], freqs)
    with pytest.raises(ValueError):
        apply_rotary(q, q[:, :, :32], pos, freqs)
    with pytest.raises(ValueError):
        apply_rotary(q, None, pos, rotary_frequencies(66, device=cuda)[0])
    with pytest.raises(ValueError):
        apply_rotary(q, None, pos[:, None].expand(4, 2), freqs, sections=(16, 15))
    with pytest.raises(ValueError):
        apply_rotary(q[0], None, pos, freqs)
    with pytest.raises(TypeError):
        apply_rotary(q, None, pos.float(), freqs)
    with pytest.raises(TypeError):
        apply_rotary(q, None, pos, freqs.float())
    with pytest.raises(TypeError):
        apply_rotary(q.double(), None, pos, freqs)
    with pytest.raises(_lib.PrismError):
        apply_rotary(q, None, pos.cpu(), freqs)
