"""The launch count's table names entry points that call() is made for, not those that the torch
extension calls by itself (no GPU needed)."""
import os

from prism_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_counted_entry_points_go_through_call():
    extension = open(os.path.join(ROOT, "prism_b200", "csrc", "torch_ops.cpp")).read()
    assert [name for name in _lib.KERNELS if f"check({name}(" in extension] == []
    assert set(_lib.KERNELS) <= set(_lib.SIGNATURES)
