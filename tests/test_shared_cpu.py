"""The entry points for sequences that share pages: what they refuse before
they touch a device."""
from __future__ import annotations

import ctypes

import pytest

from pa_b200 import _lib

BAD = _lib.PA_ERR_INVALID_ARGUMENT
ONE = (ctypes.c_void_p * 1)(16)
NONE = (ctypes.c_void_p * 1)(None)
P = ctypes.c_void_p(16)


@pytest.mark.parametrize("args,want", [
    ((ONE, ONE, 17, P, P, None, 1, 1, 2, 64, 16, 8), _lib.PA_ERR_DTYPE),
    ((ONE, ONE, 1, P, P, None, -1, 1, 2, 64, 16, 8), BAD),
    ((ONE, ONE, 1, P, P, None, 1, 1, 0, 64, 16, 8), BAD),
    ((ONE, ONE, 1, P, P, None, 1, 1, 2, 64, 0, 8), BAD),
    ((ONE, ONE, 1, None, P, None, 1, 1, 2, 64, 16, 8), BAD),
    ((ONE, ONE, 1, P, None, None, 1, 1, 2, 64, 16, 8), BAD),
    ((None, ONE, 1, P, P, None, 1, 1, 2, 64, 16, 8), BAD),
    ((NONE, ONE, 1, P, P, None, 1, 1, 2, 64, 16, 8), BAD),
    ((None, None, 1, None, None, None, 0, 1, 2, 64, 16, 8), _lib.PA_OK),
    ((None, None, 1, P, P, None, 3, 0, 2, 64, 16, 8), _lib.PA_OK),
])
def test_copy_blocks(args, want):
    assert _lib.call("pa_copy_blocks", *args, None, None) == want


def test_remap_block_tables():
    assert _lib.call("pa_remap_block_tables", P, P, P, -1, 4, None) == BAD
    assert _lib.call("pa_remap_block_tables", None, P, P, 1, 4, None) == BAD
    assert _lib.call("pa_remap_block_tables", P, P, None, 1, 4, None) == BAD
    assert _lib.call("pa_remap_block_tables", None, None, None, 0, 4, None) == _lib.PA_OK


def _append(io=2, kv=2, T=1, seqs=1, rot=64, D=64, q=P, pos=P, cs=P, seq=P, wdt=0, H=2, BS=16):
    return _lib.call("pa_qk_norm_rope_append", P, q, 128, 64, P, 64, 64, P, 64, 64, io, P, P, wdt, 1e-6, cs, 10, rot,
                     0, pos, seq, T, P, P, kv, None, None, P, seqs, H, 1, D, BS, 8, 4, None, None)


@pytest.mark.parametrize("kw,want", [
    ({"T": -1}, BAD), ({"H": 0}, BAD), ({"BS": 0}, BAD), ({"rot": 63}, BAD), ({"rot": 66}, BAD), ({"rot": -2}, BAD),
    ({"D": 96}, _lib.PA_ERR_HEAD_DIM), ({"io": 3}, _lib.PA_ERR_DTYPE), ({"io": 4}, _lib.PA_ERR_DTYPE),
    ({"kv": 9}, _lib.PA_ERR_DTYPE), ({"wdt": 1}, _lib.PA_ERR_DTYPE), ({"T": 2, "seq": None}, BAD),
    ({"q": None}, BAD), ({"pos": None}, BAD), ({"cs": None}, BAD), ({"T": 0, "q": None}, _lib.PA_OK),
])
def test_qk_norm_rope_append(kw, want):
    assert _append(**kw) == want


def _shared(q=P, kv=1, io=1, B=3, NG=1, H=8, HKV=2, D=64, BS=16, gs=P, pl=P, ctx=P):
    return _lib.call("pa_paged_attention_shared", P, None, q, io, P, P, kv, P, ctx, gs, pl, B, NG, H, HKV, D, BS, 8, 4,
                     0.125, None, 0, None, None)


@pytest.mark.parametrize("kw,want", [
    ({"B": -1}, BAD), ({"NG": -1}, BAD), ({"H": 0}, BAD), ({"H": 9}, _lib.PA_ERR_NUM_HEADS),
    ({"D": 96}, _lib.PA_ERR_HEAD_DIM), ({"kv": 0, "io": 0}, _lib.PA_ERR_DTYPE), ({"kv": 4}, _lib.PA_ERR_DTYPE),
    ({"io": 2}, _lib.PA_ERR_DTYPE), ({"BS": 0}, BAD), ({"q": None}, BAD), ({"ctx": None}, BAD), ({"gs": None}, BAD),
    ({"pl": None}, BAD), ({"q": ctypes.c_void_p(18)}, _lib.PA_ERR_ALIGNMENT), ({"BS": 1 << 31}, _lib.PA_ERR_TOO_LARGE),
    ({"B": 1 << 32}, _lib.PA_ERR_TOO_LARGE), ({"B": 0, "q": None}, _lib.PA_OK),
])
def test_paged_attention_shared(kw, want):
    assert _shared(**kw) == want


def test_shared_workspace_size():
    n = ctypes.c_size_t(7)
    size = lambda *a: _lib.call("pa_shared_workspace_size", *a, ctypes.byref(n))  # noqa: E731
    assert size(0, 0, 8, 2, 64, 1) == _lib.PA_OK and n.value == 0
    assert size(3, 1, 9, 2, 64, 1) == _lib.PA_ERR_NUM_HEADS
    assert size(3, 1, 8, 2, 64, 3) == _lib.PA_ERR_DTYPE
    assert _lib.call("pa_shared_workspace_size", 3, 1, 8, 2, 64, 1, None) == BAD
