"""Gradient clipping's C entry looks at the lists' memory before any CUDA call: outputs that overlap a
gradient or each other are refused (no GPU needed: the addresses are never read)."""
import ctypes

import pytest

from prism_b200 import _lib

BF16, FP16, FP32 = 0, 1, 2
SIZE = {BF16: 2, FP16: 2, FP32: 4}


def _call(grads, outs, sizes, types, max_norm=1.0):
    n = len(grads)
    L = _lib.load()
    status = L.prism_clip_grad_norm((ctypes.c_void_p * n)(*grads), (ctypes.c_void_p * n)(*outs),
                                    (ctypes.c_int64 * n)(*sizes), (ctypes.c_int * n)(*types), n, _lib._F(max_norm),
                                    ctypes.c_void_p(0x1000), ctypes.c_void_p(0x2000), None)
    return status, L.prism_last_error().decode()


A = 0x7f0000000000


@pytest.mark.parametrize("name,grads,outs,sizes,types", [
    ("in place, the second inside the first", [A, A + 40], [A, A + 40], [100, 10], [FP32, FP32]),
    ("in place, one element shared", [A, A + 396], [A, A + 396], [100, 100], [FP32, FP32]),
    ("in place, the other order", [A + 396, A], [A + 396, A], [100, 100], [FP32, FP32]),
    ("in place, the same start, other lengths", [A, A], [A, A], [100, 99], [FP32, FP32]),
    ("in place, the same memory as another type", [A, A], [A, A], [100, 100], [BF16, FP16]),
    ("one output for two gradients", [A, A + 400], [A + 4096, A + 4096], [100, 100], [FP32, FP32]),
    ("outputs that overlap", [A, A + 400], [A + 4096, A + 4496 - 2], [100, 100], [FP32, FP32]),
    ("an output inside its own gradient", [A], [A + 4], [100], [FP32]),
    ("an output on the next gradient", [A, A + 400], [A + 400, A + 4096], [100, 100], [FP32, FP32]),
    ("an output on a gradient that is clipped in place", [A, A + 400], [A, A + 200], [100, 100], [FP32, FP32]),
    ("a gradient that is clipped in place is read, too", [A, A], [A, A + 4096], [100, 100], [FP32, FP32]),
    ("the last of many", [A + 512 * i for i in range(300)], [A + 512 * i for i in range(299)] + [A + 512 * 7 + 256],
     [128] * 300, [FP32] * 300),
])
@pytest.mark.parametrize("flipped", [False, True])
def test_refused(name, grads, outs, sizes, types, flipped):
    if flipped:
        grads, outs, sizes, types = (v[::-1] for v in (grads, outs, sizes, types))
    status, message = _call(grads, outs, sizes, types)
    assert status == 1 and "overlap" in message, (name, status, message)
