"""Forward-mode derivatives, which the operators around the attention do not have, are refused, not left
out."""
import pytest
import torch
from torch.autograd import forward_ad

from prism_b200 import add_rms_norm, add_rms_norm_fp8, apply_rotary, linear_fp8, quantize_rows_fp8, rotary_frequencies

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode(requires_grad, cuda):
    x, w = torch.randn(3, 64, device=cuda), torch.ones(64, device=cuda)
    q, pos = torch.randn(3, 2, 64, device=cuda), torch.arange(3, device=cuda)
    freqs, _ = rotary_frequencies(64, device=cuda)
    x8, xs = quantize_rows_fp8(x)
    b = torch.zeros(3, device=cuda)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t.clone().requires_grad_() if requires_grad else t, torch.ones_like(t))
        calls = [lambda: add_rms_norm(dual(x)), lambda: add_rms_norm(x, dual(x)), lambda: add_rms_norm(x, x, dual(w)),
                 lambda: apply_rotary(dual(q), None, pos, freqs), lambda: apply_rotary(q, dual(q), pos, freqs),
                 lambda: apply_rotary(q, q, pos, dual(freqs)),
                 lambda: add_rms_norm_fp8(dual(x)), lambda: add_rms_norm_fp8(x, dual(x)),
                 lambda: add_rms_norm_fp8(x, x, dual(w)), lambda: quantize_rows_fp8(dual(x)),
                 lambda: linear_fp8(x8, dual(xs), x8, xs), lambda: linear_fp8(x8, xs, x8, dual(xs)),
                 lambda: linear_fp8(x8, xs, x8, xs, dual(b))]
        for call in calls:
            with pytest.raises(NotImplementedError):
                call()
        # the same tensors without a tangent, inside the level
        add_rms_norm(x, x, w), apply_rotary(q, q, pos, freqs), linear_fp8(x8, xs, x8, xs, b)
