"""What the packed attention and the paged cache check on the host (no GPU needed)."""
import ctypes

import pytest
import torch

import prism_b200
from prism_b200 import _lib, append_paged, packed_attention, paged_attention

BF16, INVALID, OK = 0, 1, 0


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def _i(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_public_names():
    for name in ("packed_attention", "append_paged", "paged_attention"):
        assert callable(getattr(prism_b200, name))


CACHE = dict(k_cache=_t(4, 16, 2, 64), v_cache=_t(4, 16, 2, 64), page_table=torch.zeros(3, 2, dtype=torch.int32), lengths=_i(1, 2, 3))


def test_cpu_tensors_are_refused():
    q, k = _t(5, 4, 64), _t(5, 2, 64)
    for call in (lambda: packed_attention(q, k, k, _i(0, 5)), lambda: append_paged(_t(3, 2, 64), _t(3, 2, 64), **CACHE),
                 lambda: paged_attention(_t(3, 4, 64), **CACHE)):
        with pytest.raises(_lib.PrismError, match="CUDA"):
            call()


@pytest.mark.parametrize("error,text,change", [
    (ValueError, r"\[T, Hq, D\]", dict(q=_t(5, 256))),
    (ValueError, r"\[T, Hq, D\]", dict(v=_t(5, 1, 64))),
    (ValueError, r"\[T, Hq, D\]", dict(q=_t(5, 4, 128))),
    (TypeError, "Float", dict(q=_t(5, 4, 64, dtype=torch.float32), k=_t(5, 2, 64, dtype=torch.float32), v=_t(5, 2, 64, dtype=torch.float32))),
    (TypeError, "Half", dict(k=_t(5, 2, 64, dtype=torch.float16))),
    (ValueError, "head dim 80", dict(q=_t(5, 4, 80), k=_t(5, 2, 80), v=_t(5, 2, 80))),
    (ValueError, "3 query heads do not share 2", dict(q=_t(5, 3, 64))),
    (ValueError, "258 query heads", dict(q=_t(5, 258, 64))),
    (ValueError, "0 query heads", dict(q=_t(5, 0, 64))),
    (TypeError, "Float", dict(offsets=torch.tensor([0.0, 5.0]))),
    (ValueError, "one row number more", dict(offsets=torch.zeros(0, dtype=torch.int32))),
    (ValueError, "one row number more", dict(offsets=torch.zeros(2, 2, dtype=torch.int32))),
    (ValueError, "shape and type of offsets", dict(k_offsets=_i(0, 1, 5))),
    (ValueError, "shape and type of offsets", dict(k_offsets=torch.tensor([0, 5]))),
    (ValueError, "without k_offsets", dict(k=_t(6, 2, 64), v=_t(6, 2, 64))),
    (ValueError, "scale", dict(scale=0.0)),
    (ValueError, "scale", dict(scale=-1.0)),
    (ValueError, "scale", dict(scale=float("nan"))),
    (ValueError, "scale", dict(scale=float("inf"))),
])
def test_packed_attention_refusals(error, text, change):
    args = dict(q=_t(5, 4, 64), k=_t(5, 2, 64), v=_t(5, 2, 64), offsets=_i(0, 5))
    with pytest.raises(error, match=text):
        packed_attention(**(args | change))


CACHE_REFUSALS = [
    (ValueError, r"\[pages, page_size, Hk, D\]", dict(k_cache=_t(4, 16, 128))),
    (ValueError, r"\[pages, page_size, Hk, D\]", dict(v_cache=_t(4, 8, 2, 64))),
    (TypeError, "Half", dict(v_cache=_t(4, 16, 2, 64, dtype=torch.float16))),
    (TypeError, "Float", dict(k_cache=_t(4, 16, 2, 64, dtype=torch.float32), v_cache=_t(4, 16, 2, 64, dtype=torch.float32))),
    (ValueError, "columns must be contiguous", dict(k_cache=_t(4, 16, 64, 2).transpose(2, 3))),
    (TypeError, "Long", dict(page_table=torch.zeros(3, 2, dtype=torch.int64))),
    (TypeError, "Long", dict(lengths=torch.tensor([1, 2, 3]))),
    (ValueError, "page_table must be", dict(page_table=torch.zeros(2, 2, dtype=torch.int32))),
    (ValueError, "page_table must be", dict(lengths=torch.zeros(3, 1, dtype=torch.int32))),
]


@pytest.mark.parametrize("error,text,change", CACHE_REFUSALS + [
    (ValueError, r"\[B, Hk, D\]", dict(k=_t(3, 1, 64))),
    (ValueError, r"\[B, Hk, D\]", dict(v=_t(3, 2, 32))),
    (ValueError, r"\[B, Hk, D\]", dict(k=_t(3, 1, 2, 64), v=_t(3, 1, 2, 64), offsets=_i(0, 1, 2, 3))),
    (TypeError, "caches' type", dict(k=_t(3, 2, 64, dtype=torch.float16))),
    (ValueError, "q must have", dict(q=_t(2, 4, 64))),
    (ValueError, "q must have", dict(q=_t(3, 4, 64, dtype=torch.float16))),
    (ValueError, "q must have", dict(q=_t(3, 1, 4, 64))),
    (ValueError, "offsets must hold", dict(offsets=_i(0, 3))),
    (TypeError, "Float", dict(offsets=torch.zeros(4))),
    (ValueError, "2 sequences of k, 3 of lengths", dict(k=_t(2, 2, 64), v=_t(2, 2, 64))),
    (ValueError, "layout", dict(layout="x")),
    (TypeError, "float64", dict(freqs=torch.zeros(32))),
    (ValueError, "33 pairs", dict(freqs=torch.zeros(33, dtype=torch.float64))),
    (ValueError, "up to 256", dict(k=_t(3, 2, 320), v=_t(3, 2, 320), k_cache=_t(4, 16, 2, 320), v_cache=_t(4, 16, 2, 320))),
])
def test_append_refusals(error, text, change):
    with pytest.raises(error, match=text):
        append_paged(**(dict(k=_t(3, 2, 64), v=_t(3, 2, 64)) | CACHE | change))


@pytest.mark.parametrize("error,text,change", CACHE_REFUSALS + [
    (ValueError, "q must be", dict(q=_t(4, 4, 64))),
    (ValueError, "q must be", dict(q=_t(3, 4, 128))),
    (ValueError, "q must be", dict(q=_t(12, 64))),
    (TypeError, "Half", dict(q=_t(3, 4, 64, dtype=torch.float16))),
    (ValueError, "head dim 32", dict(q=_t(3, 4, 32), k_cache=_t(4, 16, 2, 32), v_cache=_t(4, 16, 2, 32))),
    (ValueError, "3 query heads do not share 2", dict(q=_t(3, 3, 64))),
    (ValueError, "scale", dict(scale=0.0)),
])
def test_paged_attention_refusals(error, text, change):
    with pytest.raises(error, match=text):
        paged_attention(**(dict(q=_t(3, 4, 64)) | CACHE | change))


def test_c_entries_refuse_bad_arguments():
    """Every refusal below comes from the host checks, before any CUDA call."""
    L = _lib.load()
    f, n = ctypes.c_float, None
    some = (ctypes.c_int64 * 3)(128, 64, 64)
    odd = (ctypes.c_int64 * 3)(132, 64, 64)
    p, off16 = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)   # never read

    def packed(q=p, qs=some, rows=4, hq=2, hk=1, D=64, scale=1.0, dtype=BF16, o=p, lse=n, rest=n, at=p, count=1):
        return L.prism_packed_attention(q, qs, p, some, p, some, at, at, 0, count, rows, rows, hq, hk, D, 1, f(scale), dtype,
                                        o, lse, rest, n, n)

    assert packed(rows=0) == OK
    for change, text in [(dict(q=n), b"null"), (dict(o=n), b"null"), (dict(at=n), b"null"), (dict(q=off16), b"16 bytes"),
                         (dict(qs=odd), b"16 bytes"), (dict(o=off16), b"32 bytes"), (dict(D=96), b"head dim"),
                         (dict(hq=3, hk=2), b"share"), (dict(hq=129), b"share"), (dict(hk=0), b"share"), (dict(scale=0.0), b"scale"),
                         (dict(scale=float("nan")), b"scale"), (dict(dtype=2), b"type"), (dict(rows=-1), b"sizes"),
                         (dict(count=-1), b"sizes"), (dict(lse=p), b"belong together"), (dict(rows=1 << 30), b"sizes"),
                         (dict(lse=p, rest=p, dtype=1), b"bf16")]:
        assert packed(**change) == INVALID, change
        assert text in L.prism_last_error(), (change, L.prism_last_error())
    bwd = lambda rows, dk=p, dv=p, ws=p: L.prism_packed_attention_bwd(
        p, some, p, some, p, some, p, p, p, some, p, p, p, 0, 1, rows, rows, 2, 1, 64, 1, f(1.0), ws, p, dk, dv, n)
    assert bwd(0) == INVALID and b"no rows" in L.prism_last_error()
    assert bwd(4, dv=n) == INVALID and bwd(4, ws=n) == INVALID and bwd(4, dk=off16) == INVALID

    def append(tokens=3, dim=64, rot=64, batch=3, page_size=16, k=p, freqs=p, table=p, dtype=BF16, heads=1, offsets=n, width=2):
        return L.prism_append_paged(n, n, 0, k, some, p, some, heads, tokens, dim, offsets, 0, batch, p, some, p, some, 4,
                                    page_size, table, 2, width, p, rot, 1, freqs, f(1.0), dtype, n, n)

    assert append(tokens=0) == OK
    for change in (dict(dim=257), dict(rot=63), dict(rot=66), dict(page_size=0), dict(k=n), dict(freqs=n), dict(table=n),
                   dict(dtype=2), dict(heads=0), dict(tokens=4), dict(tokens=-1), dict(width=1 << 27), dict(batch=0)):
        assert append(**change) == INVALID, change

    def paged(batch=3, tokens=1, hq=2, hk=1, D=64, q=p, cache=p, strides=some, scale=1.0, dtype=BF16, o=p, page_size=16, pages=4):
        return L.prism_paged_attention(q, some, batch, tokens, hq, hk, D, cache, strides, cache, strides, pages, page_size, p, 2,
                                       2, p, f(scale), dtype, o, n, n)

    assert paged(batch=0) == OK and paged(tokens=0) == OK
    far = (ctypes.c_int64 * 3)(1 << 34, 64, 64)
    for change in (dict(D=96), dict(hq=3, hk=2), dict(q=n), dict(o=n), dict(cache=n), dict(cache=off16), dict(strides=odd),
                   dict(strides=far), dict(scale=0.0), dict(dtype=2), dict(batch=1 << 28), dict(page_size=512)):
        assert paged(**change) == INVALID, change


def test_workspaces():
    """Parts where there are few tiles and long keys, none where a wave of them is full."""
    L = _lib.load()
    none = L.prism_packed_attention_workspace_bytes
    assert none(1 << 20, 1 << 20, 1, 32, 8, 128) == 0          # many tiles
    assert none(100, 100, 1, 32, 8, 128) == 0                  # short keys
    parts = none(100, 100000, 1, 32, 8, 128) / (100 * 32 * (128 * 4 + 8))
    assert parts == int(parts) and 2 <= parts <= 16
    assert L.prism_paged_attention_workspace_bytes(128, 16, 32) == 0
    assert L.prism_paged_attention_workspace_bytes(128, 16, 33) > 0
    stats = L.prism_packed_attention_stats_bytes(1000, 3, 8, 2)
    assert stats >= 1000 * 8 * 4
    assert L.prism_packed_attention_bwd_workspace_bytes(1000, 1000, 3, 8, 2, 64) >= stats
