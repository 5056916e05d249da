"""pa_paged_attention_shared on batches whose prefixes go to the tensor cores.

Every batch here is checked to be one: the work that make_plan counts for the
tensor memory has to pass its threshold on the SMs that the device has.
Tolerances are those of test_shared_gpu, whose plain form in 64 bits is used."""
from __future__ import annotations

import ctypes

import pytest
import torch

from abi_helpers import ptr, stream
from pa_b200 import _lib
from test_shared_gpu import DT, formula, make, near

pytestmark = pytest.mark.gpu


def in_tensor_memory(groups, G, HKV):
    """Whether prefixes of `groups` ((members, usable prefix), ...) go to the tensor memory: groups of 33 rows
    or more count ceil(rows / 256) units a KV head of ceil(prefix / 64) + 6 tiles, 6 tiles per SM are needed."""
    tiles = sum(HKV * -(-n * G // 256) * (-(-prefix // 64) + 6) for n, prefix in groups if n * G >= 33 and prefix)
    return tiles >= 6 * torch.cuda.get_device_properties(0).multi_processor_count


def call(q, kc, vc, bt, ctx, gs, pl, scale, offset=0):
    """Through the C ABI: (out, lse, the device's status).  The workspace starts `offset` bytes past a 512-byte
    boundary; what lies around it has to stay."""
    B, H, D = q.shape
    NB, BS, HKV, _ = kc.shape
    NG = pl.numel()
    n = ctypes.c_size_t()
    _lib.check("ws", _lib.call("pa_shared_workspace_size", B, NG, H, HKV, D, DT[q.dtype], ctypes.byref(n)))
    room = torch.full((n.value + 2 * 512,), 0xa5, dtype=torch.uint8, device="cuda")
    assert room.data_ptr() % 512 == 0
    ws = room[offset:offset + n.value]
    out, lse = torch.empty_like(q), torch.empty((B, H), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _lib.check("shared", _lib.call("pa_paged_attention_shared", ptr(out), ptr(lse), ptr(q), DT[q.dtype], ptr(kc),
                                   ptr(vc), DT[q.dtype], ptr(bt), ptr(ctx), ptr(gs), ptr(pl), B, NG, H, HKV, D, BS, NB,
                                   bt.shape[1], scale, ptr(ws), n.value, ptr(status), stream()))
    assert bool((room[:offset] == 0xa5).all()) and bool((room[offset + n.value:] == 0xa5).all())
    return out, lse, int(status)


def check(args, scale=None, status=0, **kw):
    q, kc, vc, bt, ctx, gs, pl = args
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, lse, got = call(*args, scale, **kw)
    assert got == status
    near(out, lse, *formula(q, kc, vc, bt, ctx, scale), q.dtype)


def equal_groups(seed, groups, members, prefixes, tail, H, HKV, D, dtype, BS=16):
    """`groups` groups of `members`, their prefixes taken in turn, own tokens from 0 to `tail`."""
    pre = [prefixes[g % len(prefixes)] for g in range(groups)]
    ctx = [p + (7 * m + 3 * g) % (tail + 1) for g, p in enumerate(pre) for m in range(members)]
    assert in_tensor_memory([(members, p) for p in pre], H // HKV, HKV)
    return make(seed, H, HKV, D, dtype, BS, list(range(0, groups * members + 1, members)), pre, ctx)


@pytest.mark.parametrize("groups,members,H,HKV", [(16, 16, 32, 8), (64, 16, 32, 8), (128, 8, 64, 8), (5, 40, 32, 32)])
@pytest.mark.parametrize("prefixes", [(1, 16, 40, 48, 63, 64), (65, 100, 128), (64, 300, 1, 65, 17, 128)])
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("tail", [3, 300])
def test_many_groups_of_short_prefixes(groups, members, H, HKV, prefixes, D, dtype, tail):
    """Units of one tile and of few in long rows: with one tile only one of the two chains has work."""
    check(equal_groups(D + tail, groups, members, prefixes, tail, H, HKV, D, dtype))


@pytest.mark.parametrize("offset", [16, 48, 240, 256])
def test_workspaces_on_any_16_byte_boundary(offset):
    check(equal_groups(1, 16, 16, (300,), 40, 32, 8, 128, torch.bfloat16), offset=offset)
    # without the tensor memory, and with the plan as a launch of its own
    check(make(2, 8, 2, 64, torch.float16, 5, [0, 3], [40], [50, 60, 70]), offset=offset)
    check(make(3, 4, 2, 64, torch.float16, 16, [0, 1100], [20], [20 + b % 9 for b in range(1100)]), offset=offset)


@pytest.mark.parametrize("prefixes", [(40, 64, 1), (300, 100)])
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_scales_of_zero(prefixes, D, dtype):
    """Every key weighs the same, also by a scale that is zero in 32 bits; NaN and infinities in Q are not lost."""
    q, kc, vc, bt, ctx, gs, pl = equal_groups(4, 17, 16, prefixes, 20, 32, 8, D, dtype)
    for scale in (0.0, -0.0, 1e-60):
        check((q, kc, vc, bt, ctx, gs, pl), scale=scale)
    q[3, 5, 7], q[20, 31, 0] = float("inf"), float("nan")
    check((q, kc, vc, bt, ctx, gs, pl), scale=0.0)


@pytest.mark.parametrize("prefix,members,D,dtype", [(300, 16, 128, torch.bfloat16), (20, 40, 64, torch.float16),
                                                    (4000, 70, 128, torch.float16)])
def test_waits_that_give_up(prefix, members, D, dtype):
    """Every tensor-memory CTA stops at its first tile: its groups' rows are NaN, those of the other sequences
    (a small group, one in none, an empty one) right; afterwards all of them are."""
    groups = 20
    starts = [g * members for g in range(groups + 1)]
    prefixes = [prefix] * groups
    n = starts[-1]
    ctx = [prefix + b % 30 for b in range(n)] + [60, 50, 90, 0]
    starts, prefixes = starts + [n + 2], prefixes + [40]
    assert in_tensor_memory([(members, prefix)] * groups, 4, 8)
    q, kc, vc, bt, ctx, gs, pl = make(members, 32, 8, D, dtype, 16, starts, prefixes, ctx)
    want, mean_abs, want_lse = formula(q, kc, vc, bt, ctx, 0.1)
    assert _lib.call("pa_set_shared_waits", 0) == 1
    try:
        out, lse, status = call(q, kc, vc, bt, ctx, gs, pl, 0.1)
    finally:
        assert _lib.call("pa_set_shared_waits", 1) == 0
    assert status == _lib.PA_DEVERR_TIMEOUT
    assert bool(out[:n].isnan().all()) and bool(lse[:n].isnan().all())
    near(out[n:], lse[n:], want[n:], mean_abs[n:], want_lse[n:], dtype)
    check((q, kc, vc, bt, ctx, gs, pl), scale=0.1)
