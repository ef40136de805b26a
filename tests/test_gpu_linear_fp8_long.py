"""One 8-bit projection of 65 ms and more on the device: longer than any wait at the kernel's end.

Every value is 0, 1/2 or 1 in e4m3 and the scales are powers of two, so that the products of a row are exact in
float32 in any order, and the output is their bf16 rounding."""
import pytest
import torch

from prism_b200 import _lib, linear_fp8

pytestmark = pytest.mark.gpu


def test_long_call(cuda):
    M, N, K = 3_600_001, 5120, 5120
    g = torch.Generator(device=cuda).manual_seed(0)
    draw = lambda rows: torch.randint(0, 3, (rows, K), generator=g, device=cuda, dtype=torch.uint8)
    code = torch.tensor([0x00, 0x30, 0x38], dtype=torch.uint8, device=cuda)     # 0, 1/2, 1
    few = code[draw(997).long()]
    x8 = torch.empty(M, K, dtype=torch.uint8, device=cuda)
    for a in range(0, M, 997):
        x8[a:a + 997] = few[:min(997, M - a)]
    w8 = code[draw(N).long()]
    as8 = lambda t: t.view(torch.float8_e4m3fn)
    xs = torch.full((M,), 0.25, device=cuda)
    xs[1::2] = 2.0
    ws = torch.full((N,), 0.5, device=cuda)
    y = linear_fp8(as8(x8), xs, as8(w8), ws)
    torch.cuda.synchronize()
    assert _lib.load().prism_device_status() == 0
    sums = as8(few).float() @ as8(w8).float().t()      # exact: multiples of 1/4 below 2^13
    for a in list(range(0, M, 997 * 400)) + [M - M % 997 - 997, M - M % 997]:
        rows = min(997, M - a)
        want = (sums[:rows] * xs[a:a + rows, None] * 0.5).to(torch.bfloat16)
        assert torch.equal(y[a:a + rows], want), a
