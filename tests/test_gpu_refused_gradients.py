"""Gradients with respect to rotary frequencies and to 8-bit operands, which the operators do not have, are
refused, not left out."""
import pytest
import torch

from prism_b200 import apply_rotary, linear_fp8, quantize_rows_fp8, rotary_frequencies

pytestmark = pytest.mark.gpu


def test_gradients_of_frequencies_and_8bit_operands(cuda):
    q, pos = torch.randn(3, 2, 64, device=cuda), torch.arange(3, device=cuda)
    freqs, _ = rotary_frequencies(64, device=cuda)
    learned = freqs.clone().requires_grad_()
    for query in (q, q.clone().requires_grad_()):
        with pytest.raises(NotImplementedError):
            apply_rotary(query, None, pos, learned)
    x8, xs = quantize_rows_fp8(torch.randn(4, 64, device=cuda))
    for a, b in ((x8.clone().requires_grad_(), x8), (x8, x8.clone().requires_grad_())):
        with pytest.raises(NotImplementedError):
            linear_fp8(a, xs, b, xs)
    with torch.no_grad():   # nothing is asked for here
        apply_rotary(q, None, pos, learned)
        linear_fp8(x8.clone().requires_grad_(), xs, x8, xs)
