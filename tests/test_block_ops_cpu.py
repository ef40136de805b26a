"""What the norm, rotary, clipping and 8-bit projection entry points check on the host, and the
scaled rotary frequencies (no GPU needed)."""
import math

import pytest
import torch

import prism_b200
from prism_b200 import _lib
from prism_b200.rotary import rotary_frequencies


def test_public_names():
    for name in ("add_rms_norm", "add_rms_norm_fp8", "quantize_rows_fp8", "apply_rotary", "rotary_frequencies",
                 "clip_grad_norm", "linear_fp8"):
        assert callable(getattr(prism_b200, name))


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 16)
    freqs, _ = rotary_frequencies(16)
    for call in (lambda: prism_b200.add_rms_norm(x, x), lambda: prism_b200.add_rms_norm_fp8(x),
                 lambda: prism_b200.quantize_rows_fp8(x), lambda: prism_b200.clip_grad_norm([x], 1.0),
                 lambda: prism_b200.apply_rotary(x.view(2, 1, 16), None, torch.arange(2), freqs),
                 lambda: prism_b200.linear_fp8(x.to(torch.float8_e4m3fn), torch.ones(2),
                                               x.to(torch.float8_e4m3fn), torch.ones(2))):
        with pytest.raises(_lib.PrismError):
            call()


def test_refusals_say_what_they_got():
    """Shapes and types in the messages, raised before any device is looked at."""
    x, pos = torch.zeros(2, 1, 16), torch.arange(2)
    freqs, _ = rotary_frequencies(16)
    f8 = lambda *s: torch.zeros(*s).to(torch.float8_e4m3fn)
    for error, text, call in [
            (ValueError, "8 columns", lambda: prism_b200.apply_rotary(x[..., :8], None, pos, freqs)),
            (ValueError, "[3]", lambda: prism_b200.apply_rotary(x, None, torch.arange(3), freqs)),
            (ValueError, "add up to 8", lambda: prism_b200.apply_rotary(x, None, pos, freqs, sections=(3, 3))),
            (ValueError, "'x'", lambda: prism_b200.apply_rotary(x, None, pos, freqs, layout="x")),
            (TypeError, "Float", lambda: prism_b200.apply_rotary(x, None, pos.float(), freqs)),
            (ValueError, "[2, 32]", lambda: prism_b200.linear_fp8(f8(2, 32), torch.ones(2), f8(2, 16), torch.ones(2))),
            (ValueError, "1 outputs", lambda: prism_b200.clip_grad_norm([x, x], 1.0, out=[x]))]:
        with pytest.raises(error) as e:
            call()
        assert text in str(e.value)


def test_c_entries_refuse_bad_arguments():
    """Every refusal below comes from the host checks, before any CUDA call."""
    L = _lib.load()
    f = lambda v: _lib._F(v)
    assert L.prism_add_rms_norm(None, 8, None, 0, None, f(1e-6), 4, 8, 0, None, None, None, None) == 1
    assert b"null pointer" in L.prism_last_error()
    assert L.prism_add_rms_norm(None, 8, None, 0, None, f(1e-6), 4, 0, 0, None, None, None, None) == 1
    assert L.prism_add_rms_norm(None, 8, None, 0, None, f(1e-6), 0, 8, 0, None, None, None, None) == 0
    assert L.prism_add_rms_norm_fp8(None, 8, None, 0, None, f(1e-6), 1, 4, 8, 0, None, None, None, None) == 1
    assert L.prism_add_rms_norm_bwd(None, 8, None, 8, None, 0, None, None, 4, 8, 0, None, None, None, None) == 1
    assert L.prism_rotary(None, None, 2, None, None, 0, 1, 4, 64, 63, 0, None, 0, None, None, None, f(1), 0, 0, None,
                          None, None, None, None) == 1
    assert L.prism_rotary(None, None, 2, None, None, 0, 1, 4, 64, 64, 0, None, 0, None, None, None, f(1), 0, 0, None,
                          None, None, None, None) == 1
    assert L.prism_clip_grad_norm(None, None, None, None, 3, f(1.0), None, None, None) == 1
    assert L.prism_linear_fp8(None, 32, None, None, 32, None, None, 4, 8, 24, None, 8, None) == 1
    assert b"multiple of 16" in L.prism_last_error()
    assert L.prism_linear_fp8(None, 32, None, None, 32, None, None, 4, 8, 32, None, 8, None) == 1
    assert L.prism_linear_fp8(None, 32, None, None, 32, None, None, 0, 8, 32, None, 8, None) == 0


def test_plain_and_linear_frequencies():
    f, gain = rotary_frequencies(64, 10000.0)
    assert f.dtype == torch.float64 and gain == 1.0
    assert all(math.isclose(float(f[j]), 10000.0 ** (-2 * j / 64), rel_tol=1e-12) for j in range(32))
    g, gain = rotary_frequencies(64, 10000.0, scaling="linear", factor=8.0)
    assert torch.allclose(g * 8, f, rtol=1e-12) and gain == 1.0


def test_ntk_frequencies():
    """The fastest pair keeps its frequency, the slowest is divided by the factor."""
    f, _ = rotary_frequencies(128, 10000.0)
    g, gain = rotary_frequencies(128, 10000.0, scaling="ntk", factor=4.0)
    assert gain == 1.0 and float(g[0]) == 1.0
    assert math.isclose(float(g[-1]) * 4, float(f[-1]), rel_tol=1e-9)


def test_yarn_frequencies():
    """Pairs that turn often over the original length are kept, slow ones interpolated, a
    monotonic mixture between."""
    length, factor = 4096, 16.0
    f, _ = rotary_frequencies(128, 10000.0)
    g, gain = rotary_frequencies(128, 10000.0, scaling="yarn", factor=factor, original_length=length)
    assert math.isclose(gain, 0.1 * math.log(factor) + 1)
    turns, ratio = f * length / (2 * math.pi), g / f
    # the ramp starts and ends at whole pairs, one inside each limit at most
    assert torch.allclose(ratio[turns > 32 * 1.2], torch.ones((), dtype=torch.float64))
    assert torch.allclose(ratio[turns < 1 / 1.2], torch.full((), 1 / factor, dtype=torch.float64))
    assert bool((ratio[1:] <= ratio[:-1] + 1e-12).all())
    same, gain = rotary_frequencies(128, 10000.0, scaling="yarn", factor=1.0, original_length=length)
    assert torch.allclose(same, f) and gain == 1.0


@pytest.mark.parametrize("args,kw", [((0,), {}), ((7,), {}), ((64,), {"scaling": "cubic"}),
                                     ((64,), {"scaling": "yarn", "factor": 2.0}), ((64,), {"factor": 0.5}),
                                     ((2,), {"scaling": "ntk", "factor": 2.0})])
def test_frequency_refusals(args, kw):
    with pytest.raises(ValueError):
        rotary_frequencies(*args, **kw)
