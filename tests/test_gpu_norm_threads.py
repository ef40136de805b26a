"""Norms of two widths from two host threads, each on its own stream: what one call asks of the
device does not depend on the other's."""
import threading

import pytest
import torch

from prism_b200.norm import add_rms_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("backward", [False, True])
def test_two_widths_at_once(backward, cuda):
    errors, outs = [], {}

    def work(cols):
        try:
            torch.cuda.set_device(cuda)
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                x = torch.full((4, cols), 2.0, device=cuda, requires_grad=backward)
                for _ in range(1500):
                    y = add_rms_norm(x)[0]
                    if backward:
                        torch.autograd.grad(y, x, y.detach())
                outs[cols] = y.detach()
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(c,)) for c in (8192, 13824)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for cols, y in outs.items():   # 2 / sqrt(4 + 1e-6), within a few units of fp32
        assert bool(((y - 1).abs() <= 1e-6).all())
