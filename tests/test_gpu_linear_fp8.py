"""8-bit projection (prism_b200.linear.linear_fp8) against float64 over the same 8-bit values:
one token to many, ragged token, feature and K counts, strides, a bias, and non-finite rows.

Bound: products of e4m3 values are exact in fp32; a sum of K of them in the tensor core is at most
K 2^-23 of the sum of magnitudes off; scales and bias add 2^-22, and bf16 rounds by half a unit in the last place."""
import pytest
import torch

from prism_b200 import _lib
from prism_b200.linear import linear_fp8
from prism_b200.norm import add_rms_norm_fp8, quantize_rows_fp8

pytestmark = pytest.mark.gpu


def _inputs(M, N, K, cuda, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=cuda) * torch.randn(K, generator=g, device=cuda).exp()
    w = torch.randn(N, K, generator=g, device=cuda) / K ** 0.5
    return (*quantize_rows_fp8(x.to(torch.bfloat16)), *quantize_rows_fp8(w),
            torch.randn(N, generator=g, device=cuda))


def _check(y, x8, xs, w8, ws, b, what=""):
    x, w = x8.float().double() * xs.double()[:, None], w8.float().double() * ws.double()[:, None]
    ref, size = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        ref, size = ref + b.double(), size + b.double().abs()
    bound = torch.finfo(torch.bfloat16).eps / 2 * ref.abs() * 1.01 + (x.shape[1] * 2.0 ** -23 + 2.0 ** -22) * size
    off = (y.double() - ref).abs()
    assert bool((off <= bound).all()), (what, float((off / bound.clamp_min(1e-300)).max()))


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 64, 100, 128, 129, 300, 1025])
@pytest.mark.parametrize("N,K", [(8, 16), (128, 128), (264, 208), (1000, 1536), (5120, 272)])
def test_sizes(M, N, K, cuda):
    x8, xs, w8, ws, b = _inputs(M, N, K, cuda, seed=M + N + K)
    for bias in (b, None):
        y = linear_fp8(x8, xs, w8, ws, bias)
        assert y.shape == (M, N) and y.dtype == torch.bfloat16
        _check(y, x8, xs, w8, ws, bias)
        assert torch.equal(y, linear_fp8(x8, xs, w8, ws, bias))
    assert _lib.load().prism_device_status() == 0


@pytest.mark.parametrize("M,N,K", [(1, 5120, 5120), (16, 13824, 5120), (48, 5120, 13824), (700, 5120, 5120),
                                   (3, 131, 5136), (2500, 1537, 1536), (9450, 5120, 1024)])
def test_layer_sizes(M, N, K, cuda):
    x8, xs, w8, ws, b = _inputs(M, N, K, cuda)
    _check(linear_fp8(x8, xs, w8, ws, b), x8, xs, w8, ws, b)
    assert _lib.load().prism_device_status() == 0


@pytest.mark.parametrize("M,N,K", [(9450, 5120, 1152), (20_001, 1000, 1168), (3001, 13_832, 2064), (76_000, 264, 1040),
                                   (5000, 5001, 1040), (10_000, 4224, 5120)])
def test_many_tiles(M, N, K, cuda):
    """More tiles than SMs at a long K: odd numbers of 128-feature halves, ragged tokens, output rows
    that allow no wide stores."""
    x8, xs, w8, ws, b = _inputs(M, N, K, cuda)
    y = linear_fp8(x8, xs, w8, ws, b)
    _check(y, x8, xs, w8, ws, b)
    assert torch.equal(y, linear_fp8(x8, xs, w8, ws, b)) and _lib.load().prism_device_status() == 0


def test_shapes_strides_and_alignment(cuda):
    x8, xs, w8, ws, b = _inputs(60, 200, 256, cuda)
    ref = linear_fp8(x8, xs, w8, ws, b)
    assert torch.equal(linear_fp8(x8.view(3, 20, 256), xs.view(3, 20), w8, ws, b), ref.view(3, 20, 200))
    assert torch.equal(linear_fp8(x8[0], xs[0], w8, ws, b), linear_fp8(x8[:1], xs[:1], w8, ws, b)[0])
    wide = torch.zeros(60, 320, dtype=torch.uint8, device=cuda)
    for at in (32, 7):   # 16-byte aligned rows, and rows that are not
        wide[:, at:at + 256] = x8.view(torch.uint8)
        assert torch.equal(linear_fp8(wide.view(torch.float8_e4m3fn)[:, at:at + 256], xs, w8, ws, b), ref)
    wt = w8.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn)
    assert torch.equal(linear_fp8(x8, xs, wt, ws, b), ref)
    assert linear_fp8(x8[:0], xs[:0], w8, ws, b).shape == (0, 200)
    assert torch.equal(linear_fp8(x8, xs, w8, ws, b.to(torch.bfloat16)),
                       linear_fp8(x8, xs, w8, ws, b.to(torch.bfloat16).float()))


def test_non_finite_rows_stay_apart(cuda):
    """A token row whose scale is NaN gives a NaN row and leaves the others as they were."""
    x = torch.randn(40, 512, generator=torch.Generator().manual_seed(3)).to(cuda)
    _, _, w8, ws, b = _inputs(1, 130, 512, cuda)
    clean = linear_fp8(*add_rms_norm_fp8(x)[:2], w8, ws, b)
    x[7, 3], x[31, 500] = float("nan"), float("inf")
    y = linear_fp8(*add_rms_norm_fp8(x)[:2], w8, ws, b)
    rows = torch.tensor([i for i in range(40) if i not in (7, 31)], device=cuda)
    assert bool(y[[7, 31]].isnan().all()) and torch.equal(y[rows], clean[rows])


def test_offsets_past_32_bits(cuda):
    M, N, K = 200_001, 11_000, 64        # 2.2e9 outputs
    x8, xs, w8, ws, b = _inputs(M, N, K, cuda)
    y = linear_fp8(x8, xs, w8, ws, b)
    for rows in (slice(0, 2), slice(M - 3, M)):
        _check(y[rows], x8[rows], xs[rows], w8, ws, b)


def test_refusals(cuda):
    x8, xs, w8, ws, b = _inputs(4, 16, 32, cuda)
    with pytest.raises(TypeError):
        linear_fp8(x8.float(), xs, w8, ws)
    with pytest.raises(TypeError):
        linear_fp8(x8, xs.double(), w8, ws)
    with pytest.raises(ValueError):
        linear_fp8(x8, xs[:3], w8, ws)
    with pytest.raises(ValueError):
        linear_fp8(x8[:, :16], xs, w8, ws)
    with pytest.raises(ValueError):
        linear_fp8(x8, xs, w8, ws, b[:3])
    with pytest.raises(_lib.PrismError):
        linear_fp8(x8[:, :24], xs, w8[:, :24], ws)      # K is not a multiple of 16
    with pytest.raises(_lib.PrismError):
        linear_fp8(x8, xs.cpu(), w8, ws)
    with pytest.raises(NotImplementedError):
        linear_fp8(x8, xs, w8, ws, b.requires_grad_())
