"""pa_paged_attention_shared against the softmax in 64 bits.

Tolerance, before any run.  With u half a unit in the last place (2^-8 bf16,
2^-11 fp16) and A = sum_j p_j |V_j| the weighted mean of |V|: rounding the
weights moves out by at most u A, rounding out by u |out|, and the fp32 work
(scores of a few units summed over D <= 256 products, exp2 to 2^-22, sums) by
less than 3e-5 A.  lse is fp32 throughout: 2e-5 + 1e-6 |lse|."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from abi_helpers import ptr, stream
from pa_b200 import _lib, ops

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DT = {torch.bfloat16: _lib.PA_DTYPE_BF16, torch.float16: _lib.PA_DTYPE_F16}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(seed, H, HKV, D, dtype, BS, starts, prefixes, ctx, q_scale=1.0, spare=3):
    """Pools, tables and queries; members of a group share whole prefix pages,
    and hold copies of the page in which the prefix ends."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    B = len(ctx)
    MB = max(1, max(-(-c // BS) for c in ctx))
    own = [0] * B
    tables = np.zeros((B, MB), np.int64)
    group = {b: i for i in range(len(prefixes)) for b in range(starts[i], starts[i + 1])}
    shared = {}
    nxt = 0
    for b in range(B):
        need = -(-ctx[b] // BS)
        full = min(prefixes[group[b]] // BS, need) if b in group else 0
        if full:
            pages = shared.setdefault(group[b], [])
            while len(pages) < full:
                pages.append(nxt)
                nxt += 1
            tables[b, :full] = pages[:full]
        own[b] = full
        for j in range(full, need):
            tables[b, j] = nxt
            nxt += 1
    NB = nxt + spare
    perm = rng.permutation(NB)
    tables = perm[tables]
    kc = torch.randn((NB, BS, HKV, D), device="cuda", generator=g).to(dtype)
    vc = torch.randn((NB, BS, HKV, D), device="cuda", generator=g).to(dtype)
    for i, p in enumerate(prefixes):
        r = p % BS
        full = p // BS
        members = [b for b in range(starts[i], starts[i + 1]) if ctx[b] >= p and r]
        for b in members[1:]:
            for t in (kc, vc):
                t[tables[b, full], :r] = t[tables[members[0], full], :r].clone()
    q = (torch.randn((B, H, D), device="cuda", generator=g) * q_scale).to(dtype)
    return q, kc, vc, ints(tables.tolist()), ints(ctx), ints(starts), ints(prefixes)


def formula(q, kc, vc, bt, ctx, scale):
    B, H, D = q.shape
    NB, BS, HKV, _ = kc.shape
    out = torch.full((B, H, D), math.nan, dtype=torch.float64, device="cuda")
    mean_abs = torch.zeros((B, H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(ctx.tolist()):
        n = min(n, bt.shape[1] * BS)
        if n <= 0:
            continue
        ids = bt[b, :-(-n // BS)].long()
        k = kc[ids].double().reshape(-1, HKV, D)[:n].repeat_interleave(H // HKV, 1)
        v = vc[ids].double().reshape(-1, HKV, D)[:n].repeat_interleave(H // HKV, 1)
        s = torch.einsum("hd,nhd->hn", q[b].double(), k) * scale
        m = s.amax(1, keepdim=True)
        e = torch.exp(s - m)
        lse[b] = m[:, 0] + e.sum(1).log()
        w = e / e.sum(1, keepdim=True)
        out[b] = torch.einsum("hn,nhd->hd", w, v)
        mean_abs[b] = torch.einsum("hn,nhd->hd", w, v.abs())
    return out, mean_abs, lse


def near(got, lse, want, mean_abs, want_lse, dtype):
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(lse.isinf(), want_lse.isinf())
    u = U[dtype]
    tol = u * (want.abs() + mean_abs) + 3e-5 * mean_abs
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() - tol).nan_to_num(0).max()))
    off = (lse.double() - want_lse).abs() > 2e-5 + 1e-6 * want_lse.abs()
    assert not bool(off.any()), float((lse.double() - want_lse).abs().nan_to_num(0).max())


def run_and_check(args, dtype, scale=None):
    q, kc, vc, bt, ctx, gs, pl = args
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = ops.paged_attention_shared(q, kc, vc, bt, ctx, gs, pl, scale)
    near(out, lse, *formula(q, kc, vc, bt, ctx, scale), dtype)
    return out, lse


def tails(prefix, extra):
    return [prefix + e for e in extra]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,HKV,D", [(12, 12, 64), (32, 8, 128), (8, 1, 128), (16, 2, 256), (6, 3, 32), (40, 1, 64),
                                     (7, 7, 128), (64, 2, 128)])
@pytest.mark.parametrize("BS", [16, 5])
def test_one_group(H, HKV, D, dtype, BS):
    ctx = tails(77, [0, 1, 16, 17, 200, 3, 64, 128, 33])
    run_and_check(make(H + D, H, HKV, D, dtype, BS, [0, 9], [77], ctx), dtype)


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 127, 128, 129, 255, 256, 257, 1000])
@pytest.mark.parametrize("members", [1, 2, 16, 33])
def test_prefix_lengths(prefix, members):
    """Prefixes that end around tiles and pages; groups of one to more rows than a tile of rows."""
    ctx = tails(prefix, [(5 * b) % 23 + (prefix == 0) for b in range(members)])
    run_and_check(make(prefix, 8, 2, 64, torch.bfloat16, 16, [0, members], [prefix], ctx), torch.bfloat16)
    run_and_check(make(prefix, 4, 2, 128, torch.float16, 16, [0, members], [prefix], ctx), torch.float16)


@pytest.mark.parametrize("H,HKV,D,dtype", [(32, 8, 128, torch.bfloat16), (12, 12, 64, torch.float16)])
def test_many_rows_and_long_prefix(H, HKV, D, dtype):
    """130 members: more query rows of a KV head than any tile holds, a prefix cut into many pieces."""
    ctx = tails(3001, [b % 37 for b in range(130)])
    run_and_check(make(1, H, HKV, D, dtype, 16, [0, 130], [3001], ctx), dtype)


def test_groups_of_all_kinds():
    """Empty groups, groups of one, sequences outside any group, idle sequences first, last and alone in a group,
    a prefix longer than its members, and one of length zero."""
    starts = [2, 2, 3, 8, 8, 12, 14, 16]
    prefixes = [50, 60, 100, 70, 90, 0, 333]
    ctx = [40, 0, 81, 0, 130, 120, 100, 101, 60, 95, 90, 0, 20, 5, 0, 0, 0, 257]
    # group 4 (sequences 8..11): member 8 has 60 tokens, so 60 of the 90 are shared
    a = make(2, 32, 8, 128, torch.bfloat16, 16, starts, [min(p, 60) if i == 4 else p for i, p in enumerate(prefixes)], ctx)
    a = a[:6] + (ints(prefixes),)
    run_and_check(a, torch.bfloat16)


def test_members_without_tokens_only():
    q, kc, vc, bt, ctx, gs, pl = make(3, 8, 8, 64, torch.float16, 16, [0, 3], [10], [20, 20, 20])
    out, lse = ops.paged_attention_shared(q, kc, vc, bt, ints([0, -4, 0]), gs, pl, 0.125)
    assert bool(out.isnan().all()) and bool((lse == -math.inf).all())


def test_no_groups_and_no_sequences():
    a = make(4, 8, 2, 64, torch.bfloat16, 16, [0], [], [1, 17, 300])
    out, lse = run_and_check(a, torch.bfloat16)
    none, none_lse = ops.paged_attention_shared(a[0][:0], *a[1:], 0.125)
    assert none.shape == (0, 8, 64) and none_lse.shape == (0, 8)


@pytest.mark.parametrize("starts", [[0, 5, 3], [-1, 2, 4], [0, 2, 99]])
def test_bad_group_starts_share_nothing(starts):
    q, kc, vc, bt, ctx, _, _ = make(5, 8, 2, 64, torch.bfloat16, 16, [0], [], [30, 40, 50, 20])
    n = ctypes.c_size_t()
    _lib.check("ws", _lib.call("pa_shared_workspace_size", 4, 2, 8, 2, 64, DT[q.dtype], ctypes.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    gs, pl = ints(starts), ints([16, 16])
    _lib.check("shared", _lib.call("pa_paged_attention_shared", ptr(out), ptr(lse), ptr(q), DT[q.dtype], ptr(kc),
                                   ptr(vc), DT[q.dtype], ptr(bt), ptr(ctx), ptr(gs), ptr(pl), 4, 2, 8, 2, 64, 16,
                                   kc.shape[0], bt.shape[1], 0.125, ptr(ws), n.value, ptr(status), stream()))
    assert int(status) == _lib.PA_DEVERR_GROUP
    near(out, lse, *formula(q, kc, vc, bt, ctx, 0.125), q.dtype)


def test_bad_block_ids_and_long_contexts_are_reported():
    q, kc, vc, bt, ctx, gs, pl = make(6, 8, 2, 64, torch.float16, 16, [0, 3], [48], [60, 70, 80])
    bt2, ctx2 = bt.clone(), ctx.clone()
    bt2[2, 4] = 1 << 20  # its own last page
    ctx2[0] = 16 * bt.shape[1] + 5
    n = ctypes.c_size_t()
    _lib.check("ws", _lib.call("pa_shared_workspace_size", 3, 1, 8, 2, 64, DT[q.dtype], ctypes.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _lib.check("shared", _lib.call("pa_paged_attention_shared", ptr(out), None, ptr(q), DT[q.dtype], ptr(kc), ptr(vc),
                                   DT[q.dtype], ptr(bt2), ptr(ctx2), ptr(gs), ptr(pl), 3, 1, 8, 2, 64, 16,
                                   kc.shape[0], bt.shape[1], 0.125, ptr(ws), n.value, ptr(status), stream()))
    assert int(status) == _lib.PA_DEVERR_BLOCK_ID | _lib.PA_DEVERR_CONTEXT
    want, mean_abs, _ = formula(q, kc, vc, bt, ctx, 0.125)
    assert bool(((out[1].double() - want[1]).abs() <= 2.0 ** -10 * mean_abs[1] + 3e-5).all())


def test_unwritten_rows_do_not_matter():
    """NaN in every pool row that no key of the batch uses, in the same pages as used ones too."""
    a = make(7, 12, 4, 64, torch.bfloat16, 16, [0, 4, 9], [37, 130], tails(37, [0, 1, 5, 20]) + tails(130, [2, 0, 70, 9, 16]))
    q, kc, vc, bt, ctx, gs, pl = a
    out, lse = run_and_check(a, torch.bfloat16)
    used = torch.zeros(kc.shape[0] * 16, dtype=torch.bool, device="cuda")
    for b, n in enumerate(ctx.tolist()):
        t = torch.arange(n, device="cuda")
        used[bt[b].long()[t // 16] * 16 + t % 16] = True
    k2, v2 = kc.clone(), vc.clone()
    k2.view(-1, 4, 64)[~used] = math.nan
    v2.view(-1, 4, 64)[~used] = math.nan
    out2, lse2 = ops.paged_attention_shared(q, k2, v2, bt, ctx, gs, pl, 0.125)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


def test_extreme_scores():
    """Scores up to several hundred (one key decides), of either sign, and scores of -inf at first or throughout."""
    a = make(8, 8, 2, 128, torch.float16, 16, [0, 5], [200], tails(200, [0, 1, 30, 64, 7]), q_scale=12.0)
    run_and_check(a, torch.float16, scale=0.9)
    run_and_check(a, torch.float16, scale=-0.9)
    run_and_check(a, torch.float16, scale=0.0)
    q, kc, vc, bt, ctx, gs, pl = a
    q = q.abs() + 0.5
    rows = bt[0, :2].long()
    kc[rows] = -math.inf  # the first 32 keys of the prefix
    run_and_check((q, kc, vc, bt, ctx, gs, pl), torch.float16, scale=0.01)
    kc[:] = -math.inf
    out, lse = ops.paged_attention_shared(q, kc, vc, bt, ctx, gs, pl, 0.01)
    assert bool(out.isnan().all()) and bool((lse == -math.inf).all())


def test_infinities_and_nan_stay_in_their_row():
    q, kc, vc, bt, ctx, gs, pl = make(9, 8, 2, 64, torch.bfloat16, 16, [0, 4], [64], tails(64, [10, 20, 30, 40]))
    want = ops.paged_attention_shared(q, kc, vc, bt, ctx, gs, pl, 0.125)
    q2, v2 = q.clone(), vc.clone()
    q2[1, 3] = math.nan
    v2[bt[2, 5].long(), 3, 1, 7] = math.inf  # token 83, sequence 2's own, KV head 1
    out, lse = ops.paged_attention_shared(q2, kc, v2, bt, ctx, gs, pl, 0.125)
    assert bool(out[1, 3].isnan().all()) and bool(lse[1, 3].isnan())
    assert bool((out[2, 4:, 7] == math.inf).all())
    out[1, 3], lse[1, 3], out[2, 4:, 7] = want[0][1, 3], want[1][1, 3], want[0][2, 4:, 7]
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_repeats_are_equal_bits_and_other_streams_too():
    a = make(10, 32, 8, 128, torch.bfloat16, 16, [0, 20, 41], [900, 33], tails(900, range(20)) + tails(33, range(60, 81)))
    want = ops.paged_attention_shared(*a[:7], 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.paged_attention_shared(*a[:7], 0.1) for _ in range(20)]
    side.synchronize()
    for out, lse in got:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_strided_inputs_and_wide_tables():
    a = make(11, 8, 2, 64, torch.float16, 16, [0, 6], [40], tails(40, [0, 5, 10, 15, 20, 25]))
    q, kc, vc, bt, ctx, gs, pl = a
    want = ops.paged_attention_shared(q, kc, vc, bt, ctx, gs, pl, 0.125)
    wide = torch.full((6, bt.shape[1] + 9), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, :bt.shape[1]] = bt
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    pool = torch.stack((kc, vc))
    got = ops.paged_attention_shared(qt, pool[0], pool[1], wide, ctx.long(), gs.long(), pl.cpu(), 0.125)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_past_32_bits():
    """A pool tensor of 2.4e9 elements with the pages at its top."""
    BS, HKV, D = 16, 8, 128
    NB = 2_400_000_000 // (BS * HKV * D)
    kc = torch.empty((NB, BS, HKV, D), dtype=torch.bfloat16, device="cuda")
    vc = torch.empty((NB, BS, HKV, D), dtype=torch.bfloat16, device="cuda")
    a = make(12, 16, 8, 128, torch.bfloat16, 16, [0, 5], [70], tails(70, [0, 3, 30, 31, 60]))
    n = a[1].shape[0]
    kc[NB - n:], vc[NB - n:] = a[1], a[2]
    want = ops.paged_attention_shared(*a[:7], 0.1)
    got = ops.paged_attention_shared(a[0], kc, vc, a[3] + (NB - n), *a[4:], 0.1)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_agrees_with_the_plain_decode():
    """The same tables through paged_attention_v3_lse, which reads every context whole (fp32 q and out)."""
    a = make(13, 32, 8, 128, torch.bfloat16, 16, [0, 12], [640], tails(640, range(0, 120, 10)))
    q, kc, vc, bt, ctx, gs, pl = a
    out, lse = ops.paged_attention_shared(q, kc, vc, bt, ctx, gs, pl, 0.0884)
    ref, ref_lse = ops.paged_attention_v3_lse(q.float(), kc, vc, bt, ctx, 0.0884, 0)
    assert float((out.float() - ref).abs().max()) < 4e-3 and float((lse - ref_lse).abs().max()) < 1e-4


def test_shim_refusals():
    q, kc, vc, bt, ctx, gs, pl = make(14, 8, 2, 64, torch.float16, 16, [0, 3], [20], [30, 30, 30])
    f = ops.paged_attention_shared
    for args, text in (((q.float(), kc, vc, bt, ctx, gs, pl), "float16"),
                       ((q.bfloat16(), kc, vc, bt, ctx, gs, pl), "both"),
                       ((q.float(), kc.float(), vc.float(), bt, ctx, gs, pl), "float16"),
                       ((q, kc, vc[:1], bt, ctx, gs, pl), "alike"),
                       ((q[:, :7], kc, vc, bt, ctx, gs, pl), "divisible"),
                       ((q[..., :32], kc, vc, bt, ctx, gs, pl), "head_dim"),
                       ((q[..., :48], kc[..., :48], vc[..., :48], bt, ctx, gs, pl), "head_dim"),
                       ((q, kc, vc, bt[:2], ctx, gs, pl), "block_tables"),
                       ((q, kc, vc, bt, ctx, gs[:1], pl), "group_starts"),
                       ((q.cpu(), kc, vc, bt, ctx, gs, pl), "CUDA")):
        with pytest.raises(RuntimeError, match=text):
            f(*args, 0.125)


def test_workspace_and_alignment_refusals():
    q, kc, vc, bt, ctx, gs, pl = make(15, 8, 2, 64, torch.float16, 16, [0, 3], [20], [30, 30, 30])
    n = ctypes.c_size_t()
    _lib.check("ws", _lib.call("pa_shared_workspace_size", 3, 1, 8, 2, 64, 1, ctypes.byref(n)))
    ws, out = torch.empty(n.value, dtype=torch.uint8, device="cuda"), torch.empty_like(q)

    def call(qp=ptr(q), w=ptr(ws), wn=n.value, nb=kc.shape[0]):
        return _lib.call("pa_paged_attention_shared", ptr(out), None, qp, 1, ptr(kc), ptr(vc), 1, ptr(bt), ptr(ctx),
                         ptr(gs), ptr(pl), 3, 1, 8, 2, 64, 16, nb, bt.shape[1], 0.125, w, wn, None, stream())

    assert call() == 0
    assert call(wn=n.value - 1) == _lib.PA_ERR_WORKSPACE and call(w=None) == _lib.PA_ERR_WORKSPACE
    assert call(qp=ptr(q) + 2) == _lib.PA_ERR_ALIGNMENT and call(w=ptr(ws) + 4) == _lib.PA_ERR_ALIGNMENT
    assert call(nb=1 << 27) == _lib.PA_ERR_TOO_LARGE


@pytest.mark.parametrize("D,BS", [(64, 16), (32, 16), (128, 4)])
def test_many_sequences_and_many_groups(D, BS):
    """More sequences, then more groups, than every CTA plans for by itself."""
    rng = np.random.default_rng(D)
    ctx = (50 + rng.integers(0, 30, 1100)).tolist()
    ctx[7] = ctx[500] = ctx[1099] = 0
    run_and_check(make(16, 4, 2, D, torch.bfloat16, BS, [3, 500, 501, 1100], [50, 20, 33], ctx), torch.bfloat16)
    starts = list(range(0, 2402, 2))
    ctx = (20 + rng.integers(0, 20, 2403)).tolist()
    run_and_check(make(17, 2, 2, D, torch.float16, BS, starts, rng.integers(0, 21, len(starts) - 1).tolist(), ctx),
                  torch.float16)


@pytest.mark.parametrize("members", [9, 32, 33, 65, 100])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_groups_in_tensor_memory(members, dtype, D):
    """Prefixes long enough for the tensor cores: units of at most 128 rows and more, last units of few rows, a
    last tile of one key, groups that the warps take beside them."""
    ctx = tails(8192 + 1, [b % 40 for b in range(members)]) + tails(31, [4, 9]) + tails(5000, [b for b in range(members)])
    starts = [0, members, members + 2, 2 * members + 2]
    run_and_check(make(members, 16, 4, D, dtype, 16, starts, [8193, 31, 5000], ctx), dtype)
    run_and_check(make(members, 16, 4, D, dtype, 32, starts, [8193, 31, 5000], ctx), dtype, scale=-0.1)
