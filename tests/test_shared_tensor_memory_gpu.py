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


def near_any(got, lse, q, kc, vc, bt, ctx, scale):
    """near() for scores of any size: a weight or an output below fp16's smallest normal number is rounded by up to
    2^-25, whatever its size; a row's sum of weights is 1 at least."""
    want, mean_abs, want_lse = formula(q, kc, vc, bt, ctx, scale)
    if got.dtype == torch.float16:
        n = ctx.view(-1, 1, 1).double()
        mean_abs = mean_abs + 2.0 ** -25 * (1 + n * vc.abs().nan_to_num(0, 0).max().double()) / 2.0 ** -11
    near(got, lse, want, mean_abs, want_lse, got.dtype)


def big(seed, D, dtype, prefixes=(200, 65, 333), **kw):
    """24 groups of 16: units of 64 rows, which the two chains share by keys; one of 80 sequences: units of 256 rows
    and of 64."""
    H, HKV, members, groups = 32, 8, 16, 24
    pre = [prefixes[g % len(prefixes)] for g in range(groups)] + [prefixes[0] + 300]
    sizes = [members] * groups + [80]
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    ctx = [p + (11 * b + 5 * g) % 50 for g, (p, n) in enumerate(zip(pre, sizes)) for b in range(n)]
    assert in_tensor_memory(list(zip(sizes, pre)), H // HKV, HKV)
    return make(seed, H, HKV, D, dtype, 16, starts, pre, ctx, **kw)


KINDS = [(128, torch.bfloat16), (64, torch.float16), (128, torch.float16), (64, torch.bfloat16)]


@pytest.mark.parametrize("D,dtype", KINDS)
@pytest.mark.parametrize("scale", [0.9, -0.9, 0.02])
def test_large_scores(D, dtype, scale):
    """One key decides, and O is rescaled in later tiles."""
    a = big(20, D, dtype, q_scale=12.0)
    out, lse, status = call(*a, scale)
    assert status == 0
    near_any(out, lse, *a[:5], scale)


@pytest.mark.parametrize("D,dtype", KINDS)
def test_scores_that_grow_along_the_prefix(D, dtype):
    """Each tile's maximum is far above the one before: every one of them moves the reference."""
    q, kc, vc, bt, ctx, gs, pl = big(21, D, dtype)
    q = q.abs() + 0.25
    kc = kc.abs() * 0.02
    for b in range(q.shape[0]):
        ids = bt[b, :-(-int(ctx[b]) // 16)].long()
        kc[ids] = (torch.arange(len(ids) * 16, device="cuda").view(len(ids), 16, 1, 1) / 16).floor().to(dtype) + \
            torch.zeros_like(kc[ids])
    out, lse, status = call(q, kc, vc, bt, ctx, gs, pl, 0.1)
    assert status == 0
    near_any(out, lse, q, kc, vc, bt, ctx, 0.1)


@pytest.mark.parametrize("D,dtype", KINDS[:2])
def test_scores_of_minus_infinity(D, dtype):
    """At first (half a tile, a tile and more), throughout a prefix, everywhere."""
    q, kc, vc, bt, ctx, gs, pl = big(22, D, dtype)
    q = q.abs() + 0.5
    for g, pages in enumerate([2, 4, 7, 1000]):
        first = int(gs[g])
        kc[bt[first, :min(pages, int(pl[g]) // 16)].long()] = -float("inf")
    check((q, kc, vc, bt, ctx, gs, pl), scale=0.01)
    kc[:] = -float("inf")
    out, lse, status = call(q, kc, vc, bt, ctx, gs, pl, 0.01)
    assert status == 0 and bool(out.isnan().all()) and bool((lse == -float("inf")).all())
    out, lse, status = call(-q, -kc, vc, bt, ctx, gs, pl, -0.01)
    assert status == 0 and bool(out.isnan().all())  # scores of +inf: inf - inf


@pytest.mark.parametrize("D,dtype", KINDS[:2])
def test_unwritten_rows(D, dtype):
    """NaN in every pool row that no key uses, rows of the prefixes' last pages among them."""
    q, kc, vc, bt, ctx, gs, pl = big(23, D, dtype)
    want = call(q, kc, vc, bt, ctx, gs, pl, 0.125)
    used = torch.zeros(kc.shape[0] * 16, dtype=torch.bool, device="cuda")
    for b, n in enumerate(ctx.tolist()):
        t = torch.arange(n, device="cuda")
        used[bt[b].long()[t // 16] * 16 + t % 16] = True
    assert not bool(used.all())
    k2, v2 = kc.clone(), vc.clone()
    k2.view(-1, 8, D)[~used] = float("nan")
    v2.view(-1, 8, D)[~used] = float("nan")
    out, lse, status = call(q, k2, v2, bt, ctx, gs, pl, 0.125)
    assert status == 0 and torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("D,dtype", KINDS[:2])
def test_nan_and_infinities_stay_in_their_rows(D, dtype):
    q, kc, vc, bt, ctx, gs, pl = big(24, D, dtype)
    want = call(q, kc, vc, bt, ctx, gs, pl, 0.125)
    q2, v2 = q.clone(), vc.clone()
    q2[5, 9] = float("nan")
    q2[400, 31, 3] = float("inf")
    v2[bt[16, 1].long(), 3, 2, 7] = float("inf")  # token 19 of group 1, KV head 2
    out, lse, status = call(q2, kc, v2, bt, ctx, gs, pl, 0.125)
    assert status == 0
    assert bool(out[5, 9].isnan().all()) and bool(lse[5, 9].isnan())
    assert bool(out[400, 31].isnan().all()) and bool(lse[400, 31].isnan())
    assert bool((out[16:32, 8:12, 7] == float("inf")).all())
    for i in (0, 1):
        got, ref = (out, lse)[i], want[i]
        got[5, 9], got[400, 31] = ref[5, 9], ref[400, 31]
    out[16:32, 8:12, 7] = want[0][16:32, 8:12, 7]
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_bad_block_ids():
    """In a group's serving row: reported, the other groups right; in a row that does not serve: not read."""
    q, kc, vc, bt, ctx, gs, pl = big(25, 128, torch.bfloat16)
    want, mean_abs, want_lse = formula(q, kc, vc, bt, ctx, 0.1)
    bad = bt.clone()
    bad[16 * 3 + 2, 0] = -1
    bad[16 * 7, 1], bad[16 * 7, 2] = -5, 1 << 20
    out, lse, status = call(q, kc, vc, bad, ctx, gs, pl, 0.1)
    assert status == _lib.PA_DEVERR_BLOCK_ID
    rest = [b for b in range(q.shape[0]) if not 16 * 7 <= b < 16 * 8]
    near(out[rest], lse[rest], want[rest], mean_abs[rest], want_lse[rest], q.dtype)


def test_equal_bits_and_other_streams():
    a = big(26, 128, torch.bfloat16)
    want = call(*a, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [call(*a, 0.1) for _ in range(10)]
    side.synchronize()
    for out, lse, status in got:
        assert status == 0 and torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("members", [33, 127, 128, 129, 255, 256, 257])
@pytest.mark.parametrize("D,dtype,BS", [(128, torch.bfloat16, 16), (64, torch.float16, 48)])
def test_rows_around_a_unit(members, D, dtype, BS):
    """One query head a KV head: units of 33 rows, of one chain's rows and of both, and one row more."""
    HKV, prefix = 16, 1500
    groups = 3
    ctx = [prefix + (b * 7) % 20 for _ in range(groups) for b in range(members)]
    assert in_tensor_memory([(members, prefix)] * groups, 1, HKV)
    check(make(members, HKV, HKV, D, dtype, BS, [members * g for g in range(groups + 1)], [prefix] * groups, ctx))


@pytest.mark.parametrize("D,dtype", KINDS[:2])
@pytest.mark.parametrize("members,groups,prefixes", [(30, 40, (100, 64, 1)), (1200, 1, (3000,)), (2, 1100, (40,))])
def test_the_plan_as_a_launch_of_its_own(D, dtype, members, groups, prefixes):
    """More sequences, or groups, than every CTA plans for by itself, with prefixes in tensor memory."""
    H, HKV = (64, 2) if groups > 1024 else (32, 8)
    assert groups * members > 1024
    check(equal_groups(27, groups, members, prefixes, 9, H, HKV, D, dtype))


def test_groups_of_all_kinds_beside_them():
    """Empty groups, groups of one, idle sequences in a large group, a prefix longer than its members, sequences in
    no group, small groups, among groups in tensor memory."""
    sizes = [16, 0, 1, 40, 3, 16, 20, 16]
    prefixes = [700, 90, 50, 900, 60, 0, 640, 800]
    starts = [2]
    for n in sizes:
        starts.append(starts[-1] + n)
    B = starts[-1] + 3
    ctx = [20, 0] + [p + (3 * b) % 30 for p, n in zip(prefixes, sizes) for b in range(n)] + [300, 0, 17]
    for b in (starts[3], starts[3] + 7, starts[4] - 1, starts[6], starts[7], starts[8] - 1):
        ctx[b] = 0
    ctx[starts[6] + 5] = 500  # shorter than its group's prefix of 640: 500 are used
    usable = [500 if p == 640 else p for p in prefixes]
    assert in_tensor_memory([(n, p) for n, p in zip(sizes, usable)], 4, 16)
    a = make(28, 64, 16, 128, torch.bfloat16, 16, starts, usable, ctx)
    a = a[:6] + (torch.tensor(prefixes, dtype=torch.int32, device="cuda"),)
    assert a[0].shape[0] == B
    check(a)
