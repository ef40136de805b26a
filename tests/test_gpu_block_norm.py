"""Residual addition + RMS norm (prism_b200.norm) against its definition in float64: forward,
8-bit rows and gradients, over types, odd widths, strides, single and no rows, rows with
non-finite values, and offsets past 32 bits.

Bounds, from the arithmetic: with ``a = (cols / 32 + 64) 2^-24`` a bound on the relative error of
any fp32 row sum of non-negative terms (at most cols / 32 + 64 roundings deep), and ``rnd`` half a
unit in the last place of the output type, |got - ref| <= rnd |ref| + a * (sum of the terms'
magnitudes) elementwise."""
import pytest
import torch

from prism_b200 import _lib
from prism_b200.norm import add_rms_norm, add_rms_norm_fp8, quantize_rows_fp8

pytestmark = pytest.mark.gpu

RND = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}  # half the least subnormal
TYPES = list(RND)
EPS = 1e-6


def _a(cols):
    return (cols / 32 + 64) * 2.0 ** -24


def _within(got, ref, slack, dtype, what):
    bound = RND[dtype] * ref.abs() * (1 + 2.0 ** -8) + TINY[dtype] + slack
    bad = (got.double() - ref).abs() > bound
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst " \
                                f"{float(((got.double() - ref).abs() / bound.clamp_min(1e-300)).max()):.3g} x the bound"


def _inputs(rows, cols, dtype, cuda, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=cuda)
    x, r = (rnd(rows, cols) * rnd(cols).exp()).to(dtype), (2 * rnd(rows, cols)).to(dtype)
    return x, r, 1 + 0.3 * rnd(cols), rnd(rows, cols).to(dtype), rnd(rows, cols).to(dtype)


def _stream64(x, r):
    return (x if r is None else (x.double() + r.double()).to(x.dtype)).double()


def _forward64(x, r, w):
    h = _stream64(x, r)
    u = 1 / (h.square().mean(-1, keepdim=True) + EPS).sqrt()
    return h, u, h * u * (1.0 if w is None else w.double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 8), (1, 5120), (37, 1536), (33, 1535), (300, 130),
                                       (4, 13824), (2, 20011), (2, 40960), (0, 64)])
@pytest.mark.parametrize("residual", [True, False])
def test_forward(rows, cols, dtype, residual, cuda):
    x, r, w, _, _ = _inputs(rows, cols, dtype, cuda)
    r = r if residual else None
    for weight in (w, None):
        y, h = add_rms_norm(x, r, weight, EPS)
        h64, _, y64 = _forward64(x, r, weight)
        assert y.dtype == dtype and h.dtype == dtype and y.shape == x.shape
        assert torch.equal(h.double(), h64)
        _within(y, y64, _a(cols) * y64.abs(), dtype, "y")
        y2, h2 = add_rms_norm(x, r, weight, EPS)
        assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [16, 24, 36, 256, 264, 512, 1000, 1024, 2048, 2056, 4096, 4100, 8192, 8200, 16384,
                                  16392])
def test_widths_at_the_limits_of_each_form(cols, dtype, cuda):
    """Widths on both sides of the places where the work is split differently (lanes to a row,
    elements to a thread, whole CTAs, shared memory), forward, 8-bit and backward, over more
    rows than one CTA takes at a time and a group's share of one row more or less."""
    rows = 1200 if cols <= 4100 else 450
    x, r, w, gy, gh = _inputs(rows, cols, dtype, cuda, seed=cols)
    x.requires_grad_(), w.requires_grad_()
    y, h = add_rms_norm(x, r, w, EPS)
    dx, dw = torch.autograd.grad((y, h), (x, w), (gy, gh))
    with torch.no_grad():
        h64, u, y64 = _forward64(x, r, w)
        assert torch.equal(h.double(), h64)
        _within(y, y64, _a(cols) * y64.abs(), dtype, "y")
        y8, s, h8 = add_rms_norm_fp8(x, r, w, EPS)
        s64 = (y64.abs().amax(-1) / 448)[:, None]
        assert torch.equal(h8, h) and bool(((s.double()[:, None] - s64).abs() <= (_a(cols) + 2.0 ** -21) * s64).all())
        v = y64 / s64
        assert bool(((y8.float().double() - v).abs() <= 2.0 ** -4 * v.abs() + 2.0 ** -10 + 2 * _a(cols) * v.abs()).all())
        g, k = gy.double(), u ** 3 / cols
        terms = g * w.double() * h64
        ref = g * w.double() * u - h64 * k * terms.sum(-1, keepdim=True) + gh.double()
        size = (g * w.double() * u).abs() + h64.abs() * k * terms.abs().sum(-1, keepdim=True) + gh.double().abs()
        _within(dx, ref, 4 * _a(cols) * size, dtype, "dx")
        each = g * h64 * u
        assert bool(((dw.double() - each.sum(0)).abs() <= ((rows + 64) * 2.0 ** -24 + _a(cols)) * each.abs().sum(0)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,width", [(0, 200), (1, 193), (8, 264)])
def test_row_strides_and_offsets(dtype, offset, width, cuda):
    """Rows of wider tensors, starting at aligned and unaligned columns; 3D inputs; zero strides."""
    cols = 184
    x, r, w, _, _ = _inputs(50, 300, dtype, cuda)
    xv, rv = x[:, offset:offset + cols], r[:, :width][:, width - cols:]
    y, h = add_rms_norm(xv, rv, w[:cols].contiguous(), EPS)
    yc, hc = add_rms_norm(xv.contiguous(), rv.contiguous(), w[:cols].contiguous(), EPS)
    _, _, y64 = _forward64(xv, rv, w[:cols])
    assert torch.equal(h, hc)
    _within(y, y64, _a(cols) * y64.abs(), dtype, "strided y")
    _within(yc, y64, _a(cols) * y64.abs(), dtype, "contiguous y")
    y3, h3 = add_rms_norm(xv.reshape(5, 10, cols), rv.reshape(5, 10, cols), w[:cols], EPS)
    assert y3.shape == (5, 10, cols) and torch.equal(h3.reshape(50, cols), h)
    one = xv[:1].expand(6, cols)
    ye, _ = add_rms_norm(one, None, None, EPS)
    assert torch.equal(ye, ye[:1].expand(6, cols))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 5120), (700, 96), (2049, 40), (130, 1535), (3, 13824),
                                       (2, 20011), (2, 40960), (0, 64)])
@pytest.mark.parametrize("residual", [True, False])
def test_gradients(rows, cols, dtype, residual, cuda):
    x, r, w, gy, gh = _inputs(rows, cols, dtype, cuda, seed=1)
    x.requires_grad_(), w.requires_grad_()
    if residual:
        r.requires_grad_()
    y, h = add_rms_norm(x, r if residual else None, w, EPS)
    outs, grads = ([y, h], [gy, gh]) if residual else ([y], [gy])
    wanted = [x, w] + ([r] if residual else [])
    dx, dw, *dr = torch.autograd.grad(outs, wanted, grads)
    with torch.no_grad():
        h64, u, _ = _forward64(x, r if residual else None, w)
        g, w64 = gy.double(), w.double()
        terms = g * w64 * h64
        k = u ** 3 / cols
        parts = [g * w64 * u, -h64 * k * terms.sum(-1, keepdim=True)] + ([gh.double()] if residual else [])
        ref = sum(parts)
        size = parts[0].abs() + h64.abs() * k * terms.abs().sum(-1, keepdim=True) + (gh.double().abs() if residual else 0)
        # 4: u enters cubed, next to the sum itself
        _within(dx, ref, 4 * _a(cols) * size, dtype, "dx")
        if residual:
            assert torch.equal(dr[0], dx)
        each = g * h64 * u
        slack = ((rows + 64) * 2.0 ** -24 + _a(cols)) * each.abs().sum(0)
        assert dw.dtype == torch.float32
        assert bool(((dw.double() - each.sum(0)).abs() <= slack).all())
    again = torch.autograd.grad(add_rms_norm(x, r if residual else None, w, EPS)[:len(outs)], wanted, grads)
    assert all(torch.equal(a, b) for a, b in zip(again, [dx, dw] + dr))


def test_gradient_against_differences(cuda):
    """<grad, v> against a central difference of the kernel's own forward, in fp32: step t
    leaves a truncation of order t^2 and a rounding noise of 2^-23 sqrt(n) / t, both below 1e-3
    of |grad| |v| / sqrt(n) at t = 1e-2 and n = 4,000."""
    x, r, w, a, b = _inputs(20, 200, torch.float32, cuda, seed=2)
    for t in (x, r, w):
        t.requires_grad_()
    y, h = add_rms_norm(x, r, w, EPS)
    grads = torch.autograd.grad((y, h), (x, r, w), (a, b))
    loss = lambda *v: sum(float((o.double() * c.double()).sum()) for o, c in zip(add_rms_norm(*v, EPS), (a, b)))
    with torch.no_grad():
        for i, g in enumerate(grads):
            gen = torch.Generator(device=cuda).manual_seed(i)
            v = torch.randn(g.shape, generator=gen, device=cuda)
            t, args = 1e-2, [x, r, w]
            moved = lambda s: [p + s * t * v if j == i else p for j, p in enumerate(args)]
            diff = (loss(*moved(1)) - loss(*moved(-1))) / (2 * t)
            got = float((g.double() * v.double()).sum())
            assert abs(diff - got) <= 1e-3 * float(g.double().norm()) * float(v.double().norm()) / v.numel() ** 0.5 \
                + 1e-2 * abs(got), (i, diff, got)


def test_unused_outputs_and_partial_gradients(cuda):
    x, r, w, gy, gh = _inputs(9, 128, torch.bfloat16, cuda)
    x.requires_grad_()
    y, h = add_rms_norm(x, r, w, EPS)
    full = torch.autograd.grad((y, h), x, (gy, torch.zeros_like(gh)))[0]
    only_y = torch.autograd.grad(add_rms_norm(x, r, w, EPS)[0], x, gy)[0]
    assert torch.equal(full, only_y)
    only_h = torch.autograd.grad(add_rms_norm(x, r, w, EPS)[1], x, gh)[0]
    assert torch.equal(only_h, gh)
    # a weight in bf16 gets its gradient in bf16; broadcast output gradients have zero strides
    wb = w.to(torch.bfloat16).requires_grad_()
    dw = torch.autograd.grad(add_rms_norm(x, r, wb, EPS)[0].sum(), wb)[0]
    assert dw.dtype == torch.bfloat16
    h64, u, _ = _forward64(x.detach(), r, w)
    each = h64 * u
    assert bool(((dw.double() - each.sum(0)).abs() <= 2.0 ** -8 * each.sum(0).abs() + 1e-4 * each.abs().sum(0)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 5120), (65, 1536), (33, 1535), (2, 20011), (2, 40960),
                                       (0, 64), (19, 1100)])
def test_8bit_rows(rows, cols, dtype, cuda):
    """|y8 - y / scale| is half a unit of e4m3: 2^-4 of the value, or 2^-10 below its normals."""
    x, r, w, _, _ = _inputs(rows, cols, dtype, cuda, seed=3)
    for residual, weight in ((r, w), (None, None)):
        y8, scale, h = add_rms_norm_fp8(x, residual, weight, EPS)
        h64, _, y64 = _forward64(x, residual, weight)
        assert y8.dtype == torch.float8_e4m3fn and scale.shape == (rows,)
        assert torch.equal(h.double(), h64)
        s64 = (y64.abs().amax(-1) / 448).clamp_min(2.0 ** -100) if rows else scale.double()
        assert bool(((scale.double() - s64).abs() <= (_a(cols) + 2.0 ** -21) * s64).all())
        v = y64 / s64[:, None]
        err = (y8.float().double() - v).abs()
        assert bool((err <= 2.0 ** -4 * v.abs() + 2.0 ** -10 + 2 * _a(cols) * v.abs()).all())
    x8, s = quantize_rows_fp8(x)
    if rows:
        ref = (x.float().abs().amax(-1) / 448).clamp_min(2.0 ** -100)
        assert bool(((s - ref).abs() <= 2.0 ** -22 * ref).all())
        v = x.double() / s.double()[:, None]
        assert bool(((x8.float().double() - v).abs() <= 2.0 ** -4 * v.abs() * (1 + 2.0 ** -18) + 2.0 ** -10).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [128, 760, 768, 776, 1531, 3000, 5120, 5112, 6144, 10000])
def test_many_rows_of_each_form(cols, dtype, cuda):
    """More rows than a launch's groups hold at once, several times over, at widths where a group
    keeps one row or two on their way: forward and 8-bit rows, with a norm and without."""
    rows = max(1500, 3000000 // cols)
    x, r, w, _, _ = _inputs(rows, cols, dtype, cuda, seed=cols + 1)
    for residual in (r, None):
        h64, _, y64 = _forward64(x, residual, w)
        y, h = add_rms_norm(x, residual, w, EPS)
        assert torch.equal(h.double(), h64)
        _within(y, y64, _a(cols) * y64.abs(), dtype, "y")
        y8, s, h8 = add_rms_norm_fp8(x, residual, w, EPS)
        s64 = y64.abs().amax(-1, keepdim=True) / 448
        assert torch.equal(h8, h) and bool(((s.double()[:, None] - s64).abs() <= (_a(cols) + 2.0 ** -21) * s64).all())
        v = y64 / s64
        assert bool(((y8.float().double() - v).abs() <= 2.0 ** -4 * v.abs() + 2.0 ** -10 + 2 * _a(cols) * v.abs()).all())
    x8, s = quantize_rows_fp8(x)
    ref = x.float().abs().amax(-1) / 448
    assert bool(((s - ref).abs() <= 2.0 ** -22 * ref).all())
    v = x.double() / s.double()[:, None]
    assert bool(((x8.float().double() - v).abs() <= 2.0 ** -4 * v.abs() * (1 + 2.0 ** -18) + 2.0 ** -10).all())


@pytest.mark.parametrize("cols", [96, 1535, 5120])
def test_rows_of_zeros_and_of_non_finite_values(cols, cuda):
    """A zero row stays zero with the least scale; a row with a NaN or an infinity has scale NaN
    and does not touch its neighbours; a row whose maximum overflows nothing stays finite."""
    x, _, w, gy, _ = _inputs(6, cols, torch.bfloat16, cuda, seed=4)
    clean8, clean_s, _ = add_rms_norm_fp8(x, None, w, EPS)
    clean, _ = add_rms_norm(x, None, w, EPS)
    bad = x.clone()
    bad[0] = 0
    bad[2, cols // 2] = float("nan")
    bad[4, 5] = float("inf")
    y8, s, _ = add_rms_norm_fp8(bad, None, w, EPS)
    assert float(s[0]) == 2.0 ** -100 and not bool(y8[0].float().any())
    assert bool(s[[2, 4]].isnan().all())
    for row in (1, 3, 5):
        assert torch.equal(y8[row].float(), clean8[row].float()) and s[row] == clean_s[row]
    y, _ = add_rms_norm(bad, None, w, EPS)
    ref = torch.nn.functional.rms_norm(bad.double(), (cols,), w.double(), EPS)
    assert torch.equal(y.isnan()[[0, 1, 2, 3, 5]], ref.isnan()[[0, 1, 2, 3, 5]]) and bool(y[2].isnan().all())
    assert bool(y[4, 5].isnan()) and torch.equal(y[[1, 3, 5]], clean[[1, 3, 5]]) and not bool(y[0].any())
    x8, s0 = quantize_rows_fp8(bad)
    assert bool(s0[[2, 4]].isnan().all()) and float(s0[0]) == 2.0 ** -100
    assert bool(s0[[1, 3, 5]].isfinite().all())


def test_8bit_rows_of_large_and_tiny_values(cuda):
    """Rows whose squares leave fp32 quantise as they stand: the scale is the maximum over 448."""
    for size in (1e25, 1e-25):
        x = (torch.randn(5, 700, generator=torch.Generator().manual_seed(6)) * size).to(cuda)
        x8, s = quantize_rows_fp8(x)
        ref = (x.double().abs().amax(-1) / 448)
        assert bool(((s.double() - ref).abs() <= 2.0 ** -22 * ref).all())
        v = x.double() / s.double()[:, None]
        assert bool(((x8.float().double() - v).abs() <= 2.0 ** -4 * v.abs() * (1 + 2.0 ** -18) + 2.0 ** -10).all())


def test_offsets_past_32_bits(cuda):
    rows, cols = 420_001, 5120          # 2.15e9 elements
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=cuda)
    x[-3:] = torch.randn(3, cols, generator=torch.Generator().manual_seed(5)).to(x)
    x[:-3] = 1.0
    y, _ = add_rms_norm(x, None, None, EPS)
    _, _, y64 = _forward64(x[-3:], None, None)
    _within(y[-3:], y64, _a(cols) * y64.abs(), torch.bfloat16, "last rows")
    assert float(y[0, 0]) == 1.0
    del y
    y8, s, _ = add_rms_norm_fp8(x, None, None, EPS)
    ref8, ref_s, _ = add_rms_norm_fp8(x[-3:].contiguous(), None, None, EPS)
    assert torch.equal(y8[-3:].float(), ref8.float()) and torch.equal(s[-3:], ref_s)


def test_another_stream(cuda):
    x, r, w, _, _ = _inputs(4000, 5120, torch.bfloat16, cuda)
    ref = add_rms_norm(x, r, w, EPS)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        doubled = x * 2
        got = add_rms_norm(doubled, r, w, EPS)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[1], (doubled.float() + r.float()).to(torch.bfloat16))
    assert torch.equal(ref[0], add_rms_norm(x, r, w, EPS)[0])


def test_refusals(cuda):
    x, r, w, _, _ = _inputs(4, 64, torch.bfloat16, cuda)
    with pytest.raises(ValueError):
        add_rms_norm(x, r[:, :32], w)
    with pytest.raises(ValueError):
        add_rms_norm(x, r.float(), w)
    with pytest.raises(ValueError):
        add_rms_norm(x, r, w[:32])
    with pytest.raises(ValueError):
        add_rms_norm(x[:, :0])
    with pytest.raises(TypeError):
        add_rms_norm(x.double())
    with pytest.raises(_lib.PrismError):
        add_rms_norm(x, r.cpu(), w)
    with pytest.raises(NotImplementedError):
        add_rms_norm_fp8(x.requires_grad_(), r, w)
