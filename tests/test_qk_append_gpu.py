"""pa_qk_norm_rope_append against the formula in 64 bits.

Tolerances, before any run.  q_out in fp32: a handful of fp32 roundings per
element (sum of squares over D <= 256 in a tree, rsqrt, two products, the turn)
at values of up to ~6: 2e-5 absolute.  16-bit outputs: half a unit in the last
place of the result, at most 2^-8 (bf16) or 2^-11 (fp16) of |y|, plus the fp32
error.  v is a conversion alone: equal bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from abi_helpers import ptr, stream
from oracle import oracle as orc
from pa_b200 import _lib, ops

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F64 = torch.float64


def formula(x, w, eps, cs, rot, interleaved):
    """x [T, H, D] in 64 bits, cs [T, rot]."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    y = x.clone()
    half = rot // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cs[:, None, i], cs[:, None, half + i]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def near(got, want, dtype):
    tol = 2e-5 + HALF_ULP[dtype] * want.abs()
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() - tol).max())


def case(seed, lens, starts, H, HKV, D, rot, dtype, pool, BS=16, fused=True, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lens)
    qkv = torch.randn((T, H + 2 * HKV, D), device="cuda", generator=g).mul(spread).to(dtype)
    if not fused:
        q, k, v = (x.contiguous() for x in qkv.split((H, HKV, HKV), 1))
    else:
        q, k, v = qkv.split((H, HKV, HKV), 1)
    pos = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, lens)] or [torch.empty(0)]).to(torch.int32).cuda()
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)] or [torch.empty(0)]).to(torch.int32).cuda()
    top = max(s + n for s, n in zip(starts, lens))
    MB = -(-top // BS)
    NB = len(lens) * MB + 3
    bt = torch.randperm(NB, generator=torch.Generator().manual_seed(seed))[:len(lens) * MB]
    bt = bt.view(len(lens), MB).to(torch.int32).cuda()
    kc = torch.full((NB, BS, HKV, D), 3.0, device="cuda").to(pool)
    vc = torch.full((NB, BS, HKV, D), 5.0, device="cuda").to(pool)
    cs = ops.rope_table(top, rot)
    w = [(1 + 0.2 * torch.randn(D, device="cuda", generator=g)) for _ in range(2)]
    return q, k, v, pos, seq, bt, kc, vc, cs, w


def flat(bt, seq, pos, BS):
    return bt.long()[seq.long(), pos.long() // BS] * BS + pos.long() % BS


NONE = torch.empty(0)


@pytest.mark.parametrize("H,HKV,D,rot", [(12, 12, 64, 64), (32, 8, 128, 128), (8, 1, 256, 256), (4, 2, 32, 32),
                                         (5, 3, 128, 64), (6, 2, 64, 6), (3, 3, 32, 0), (4, 4, 256, 20)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,pool", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                        (torch.float32, torch.float16), (torch.bfloat16, torch.float64)])
@pytest.mark.parametrize("norm", [True, False])
def test_against_the_formula(H, HKV, D, rot, interleaved, dtype, pool, norm):
    q, k, v, pos, seq, bt, kc, vc, cs, w = case(D + rot, [1, 37, 16], [500, 3, 0], H, HKV, D, rot, dtype, pool)
    w = [x.to(dtype) for x in w] if norm else [NONE, NONE]
    out = ops.qk_norm_rope_append(q, k, v, w[0], w[1], 1e-5, cs, interleaved, pos, seq, kc, vc, bt, NONE, NONE)
    rows = cs[pos.long()].double()
    args = (1e-5, rows, rot, interleaved)
    near(out, formula(q.to(F64), w[0].to(F64) if norm else None, *args), dtype)
    at = flat(bt, seq, pos, 16)
    near(kc.view(-1, HKV, D)[at], formula(k.to(F64), w[1].to(F64) if norm else None, *args),
         pool if pool in HALF_ULP else torch.float32)
    assert torch.equal(vc.view(-1, HKV, D)[at], v.to(torch.float32).to(pool))
    # every other row of the pool is as it was
    rest = torch.ones(kc.shape[0] * 16, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert bool((kc.view(-1, HKV, D)[rest] == 3).all()) and bool((vc.view(-1, HKV, D)[rest] == 5).all())


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("offset", [0, 1])
def test_strides_alignment_and_block_size(fused, offset):
    """q / k / v as odd slices of larger buffers, fp32 weights, pages of 7 tokens."""
    H, HKV, D = 3, 2, 64
    q, k, v, pos, seq, bt, kc, vc, cs, w = case(7, [9, 2], [0, 60], H, HKV, D, 64, torch.float16, torch.float16,
                                                BS=7, fused=fused)
    wide = [torch.zeros((x.shape[0], x.shape[1] + 1, D + 3), dtype=x.dtype, device="cuda") for x in (q, k, v)]
    parts = [b[:, :x.shape[1], offset:offset + D] for b, x in zip(wide, (q, k, v))]
    for part, x in zip(parts, (q, k, v)):
        part.copy_(x)
    out = ops.qk_norm_rope_append(*parts, w[0], w[1], 1e-6, cs, False, pos, seq, kc, vc, bt, NONE, NONE)
    rows = cs[pos.long()].double()
    near(out, formula(q.to(F64), w[0].to(F64), 1e-6, rows, 64, False), torch.float16)
    at = flat(bt, seq, pos, 7)
    near(kc.view(-1, HKV, D)[at], formula(k.to(F64), w[1].to(F64), 1e-6, rows, 64, False), torch.float16)
    assert torch.equal(vc.view(-1, HKV, D)[at], v)
    # head_dim itself strided, and heads in reverse memory order
    t = q.transpose(1, 2).contiguous().transpose(1, 2)
    again = ops.qk_norm_rope_append(t, k, v, w[0], w[1], 1e-6, cs, False, pos, seq, kc, vc, bt, NONE, NONE)
    assert torch.equal(again, out)


def test_fp8_pool_with_scales():
    H, HKV, D = 8, 4, 64
    q, k, v, pos, seq, bt, kc, vc, cs, w = case(8, [21], [11], H, HKV, D, 64, torch.float32, torch.float32)
    kc, vc = (torch.zeros(kc.shape, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ks = torch.tensor([0.01, 0.02, 0.5, 1.0], device="cuda")
    vs = torch.tensor([0.03, 0.001, 0.25, 2.0], device="cuda")
    out = ops.qk_norm_rope_append(q, k, v, w[0], w[1], 1e-6, cs, False, pos, seq, kc, vc, bt, ks, vs)
    rows = cs[pos.long()].double()
    near(out, formula(q.to(F64), w[0].to(F64), 1e-6, rows, 64, False), torch.float32)
    at = flat(bt, seq, pos, 16)
    got_v = vc.view(torch.uint8).view(-1, HKV, D)[at].cpu().numpy()
    assert np.array_equal(got_v, orc.quantize_e4m3(v.cpu().numpy(), vs.cpu().numpy()[None, :, None]))
    # k: the formula's value, clamped to the type's range, within half a step (2^-4 of it, 2^-10 near zero)
    want = (formula(k.to(F64), w[1].to(F64), 1e-6, rows, 64, False) / ks[:, None]).clamp(-448, 448)
    got = kc.view(-1, HKV, D)[at].to(F64)
    assert bool(((got - want).abs() <= want.abs() / 16 + 2.0 ** -10 + 1e-4).all())


def test_padding_and_bad_places():
    H, HKV, D = 2, 1, 64
    q, k, v, pos, seq, bt, kc, vc, cs, w = case(9, [8], [0], H, HKV, D, 64, torch.bfloat16, torch.bfloat16, BS=4)
    pos = torch.tensor([0, -1, 1, 8, 9, 2, 3, 5], dtype=torch.int32, device="cuda")
    seq = torch.tensor([0, 0, 0, 0, 0, 7, -1, 0], dtype=torch.int32, device="cuda")
    bt[0, 1] = 99  # position 5
    cs = ops.rope_table(9, 64)  # position 9 has no row; position 8 has no page
    before = kc.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty((8, H, D), dtype=torch.bfloat16, device="cuda")
    wq, wk = (x.to(torch.bfloat16) for x in w)
    _lib.check("append", _lib.call(
        "pa_qk_norm_rope_append", ptr(out), ptr(q), q.stride(0), q.stride(1), ptr(k), k.stride(0), k.stride(1),
        ptr(v), v.stride(0), v.stride(1), _lib.PA_DTYPE_BF16, ptr(wq), ptr(wk), _lib.PA_DTYPE_BF16, 1e-6, ptr(cs),
        9, 64, 0, ptr(pos), ptr(seq), 8, ptr(kc), ptr(vc), _lib.PA_DTYPE_BF16, None, None, ptr(bt), 1, H, HKV, D, 4,
        kc.shape[0], bt.shape[1], ptr(status), stream()))
    assert int(status) == _lib.PA_DEVERR_CONTEXT | _lib.PA_DEVERR_BLOCK_ID
    assert bool((out[1] == 0).all()) and bool(out[4].isnan().all())
    fine = [0, 2, 3, 5, 6, 7]
    rows = cs[pos.long().clamp(0, 8)].double()
    want = formula(q.to(F64), wq.to(F64), 1e-6, rows, 64, False)
    near(out[fine], want[fine], torch.bfloat16)
    at = flat(bt, torch.zeros(2, dtype=torch.int32, device="cuda"), pos[[0, 2]], 4)
    rest = torch.ones(kc.shape[0] * 4, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert torch.equal(kc.view(-1, HKV, D)[rest], before.view(-1, HKV, D)[rest])
    assert not torch.equal(kc.view(-1, HKV, D)[at], before.view(-1, HKV, D)[at])


def test_one_token_per_sequence_zero_tokens_and_a_side_stream():
    H, HKV, D = 4, 2, 128
    q, k, v, pos, seq, bt, kc, vc, cs, w = case(10, [1] * 5, [3, 9, 0, 31, 16], H, HKV, D, 128, torch.bfloat16,
                                                torch.bfloat16)
    a = ops.qk_norm_rope_append(q, k, v, w[0], w[1], 1e-6, cs, True, pos, seq, kc, vc, bt, NONE, NONE)
    k1, v1 = kc.clone(), vc.clone()
    kc.fill_(3), vc.fill_(5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = ops.qk_norm_rope_append(q, k, v, w[0], w[1], 1e-6, cs, True, pos, NONE, kc, vc, bt, NONE, NONE)
    side.synchronize()
    assert torch.equal(a, b) and torch.equal(k1, kc) and torch.equal(v1, vc)
    out = ops.qk_norm_rope_append(q[:0], k[:0], v[:0], w[0], w[1], 1e-6, cs, True, pos[:0], NONE, kc, vc, bt, NONE,
                                  NONE)
    assert out.shape == (0, H, D) and torch.equal(k1, kc)


def test_large_rows_and_values():
    """Zero heads (eps alone), large values, and infinities that stay in their head."""
    H, HKV, D = 4, 1, 64
    q, k, v, pos, seq, bt, kc, vc, cs, w = case(11, [3], [100], H, HKV, D, 64, torch.bfloat16, torch.float32)
    q, k, v = q.clone(), k.clone(), v.clone()
    q[0, 0] = 0
    q[0, 1] *= 1e15
    q[1, 2, 5] = float("inf")
    k[2, 0, 3] = float("nan")
    v[2, 0, 3] = float("-inf")
    out = ops.qk_norm_rope_append(q, k, v, w[0], w[1], 1e-6, cs, False, pos, seq, kc, vc, bt, NONE, NONE)
    assert bool((out[0, 0] == 0).all())
    want = formula(q.to(F64), w[0].to(F64), 1e-6, cs[pos.long()].double(), 64, False)
    for t, h in ((0, 1), (0, 2), (1, 1), (2, 2)):
        near(out[t:t + 1, h:h + 1], want[t:t + 1, h:h + 1], torch.bfloat16)
    assert bool(out[1, 2, 5].isnan())
    at = flat(bt, seq, pos, 16)
    assert bool(kc.view(-1, D)[at[2]].isnan().all()) and not bool(kc.view(-1, D)[at[:2]].isnan().any())
    assert float(vc.view(-1, D)[at[2], 3]) == float("-inf")


def test_shim_refusals():
    q, k, v, pos, seq, bt, kc, vc, cs, w = case(12, [3], [0], 4, 2, 64, 64, torch.bfloat16, torch.bfloat16)
    ok = dict(q=q, k=k, v=v, wq=w[0], wk=w[1], cs=cs, pos=pos, seq=seq, kc=kc, vc=vc, bt=bt, ks=NONE)

    def call(**kw):
        a = {**ok, **kw}
        return ops.qk_norm_rope_append(a["q"], a["k"], a["v"], a["wq"], a["wk"], 1e-6, a["cs"], False, a["pos"],
                                       a["seq"], a["kc"], a["vc"], a["bt"], a["ks"], NONE)

    call()
    for kw, text in (({"q": q.double()}, "float32, float16"), ({"k": k[:2]}, "must be \\[T, HKV, D\\]"),
                     ({"k": k.half()}, "q's type"), ({"wq": w[0][:5]}, "weights"), ({"pos": pos[:2]}, "positions"),
                     ({"seq": seq[:2]}, "seq_ids"), ({"seq": NONE}, "row per token"),
                     ({"kc": kc.transpose(0, 1)}, "alike|contiguous"), ({"cs": cs.half()}, "cos_sin"),
                     ({"cs": ops.rope_table(50, 66)}, "invalid"), ({"ks": torch.ones(3)}, "scales"),
                     ({"q": q[..., :48], "k": k[..., :48], "v": v[..., :48]}, "head_dim")):
        with pytest.raises(RuntimeError, match=text):
            call(**kw)


@pytest.mark.parametrize("H,HKV,D,lens", [(8, 1, 128, [700, 1]), (16, 2, 64, [601, 60]), (32, 8, 128, [640]),
                                          (4, 4, 256, [593, 7]), (30, 3, 32, [900])])
def test_many_tokens(H, HKV, D, lens):
    """Enough tokens that a CTA takes whole tokens, one or two: padding among them, an odd count."""
    q, k, v, pos, seq, bt, kc, vc, cs, w = case(13, lens, [9, 40][:len(lens)], H, HKV, D, D, torch.bfloat16,
                                                torch.bfloat16)
    w = [x.to(torch.bfloat16) for x in w]
    pos[5] = -1
    out = ops.qk_norm_rope_append(q, k, v, w[0], w[1], 1e-6, cs, False, pos, seq, kc, vc, bt, NONE, NONE)
    live = pos >= 0
    rows = cs[pos[live].long()].double()
    near(out[live], formula(q[live].to(F64), w[0].to(F64), 1e-6, rows, D, False), torch.bfloat16)
    at = flat(bt, seq[live], pos[live], 16)
    near(kc.view(-1, HKV, D)[at], formula(k[live].to(F64), w[1].to(F64), 1e-6, rows, D, False), torch.bfloat16)
    assert torch.equal(vc.view(-1, HKV, D)[at], v[live]) and bool((out[5] == 0).all())
