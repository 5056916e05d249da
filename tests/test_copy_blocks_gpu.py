"""Page copies, table rewrites and the allocator's forks and compactions: the
pool after each must equal, byte for byte, what indexing on the host gives."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from abi_helpers import ptr, stream
from pa_b200 import _lib, ops
from pa_b200.kv import KVConfig, ModelConfig, TorchBlockAllocator

pytestmark = pytest.mark.gpu

INT = {1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}


def bits(t):
    return t.view(INT[t.element_size()])


def make_pool(L, NB, BS, H, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(0, 256, (L, 2, NB, BS, H, D * torch.empty(0, dtype=dtype).element_size()),
                      dtype=torch.uint8, generator=g)
    return x.cuda().view(dtype)


def layers(pool):
    return [pool[i, 0] for i in range(len(pool))], [pool[i, 1] for i in range(len(pool))]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def expected(pool, src, dst, rows, NB):
    want = bits(pool).clone()
    old = bits(pool)
    BS = pool.shape[3]
    for i, (a, b) in enumerate(zip(src, dst)):
        if not (0 <= a < NB and 0 <= b < NB):
            continue
        r = BS if rows is None else min(max(rows[i], 0), BS)
        want[:, :, b, :r] = old[:, :, a, :r]
    return want


@pytest.mark.parametrize("L,NB,BS,H,D,dtype", [
    (1, 8, 16, 1, 32, torch.float16),
    (12, 40, 16, 12, 64, torch.float16),
    (3, 33, 7, 5, 80, torch.bfloat16),
    (2, 20, 16, 8, 128, torch.float32),
    (2, 20, 1, 2, 256, torch.float64),
    (2, 20, 32, 2, 64, torch.float8_e4m3fn),
    (70, 12, 16, 2, 32, torch.bfloat16),     # two launches
    (2, 12, 3, 1, 5, torch.float16),         # rows of 10 bytes
    (2, 12, 4, 1, 3, torch.float8_e4m3fn),   # rows of 3 bytes
])
@pytest.mark.parametrize("partial", [False, True])
def test_copies_equal_indexing(L, NB, BS, H, D, dtype, partial):
    pool = make_pool(L, NB, BS, H, D, dtype)
    perm = np.random.default_rng(1).permutation(NB).tolist()
    n = NB // 2
    src = [perm[n + i // 2] for i in range(n)]  # some pages copied twice
    dst = perm[:n]
    rows = [i % (BS + 3) - 1 for i in range(n)] if partial else None  # below 0 and above BS too
    want = expected(pool, src, dst, rows, NB)
    k, v = layers(pool)
    ops.copy_blocks(k, v, ints(src), ints(dst), ints(rows) if partial else torch.empty(0))
    assert torch.equal(bits(pool), want)


def test_bad_ids_are_skipped_and_reported():
    pool = make_pool(2, 6, 4, 2, 8, torch.float16)
    src, dst = [0, -1, 1, 9, 2], [3, 4, 6, 5, 2]
    want = expected(pool, src, dst, None, 6)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = layers(pool)
    kp = (ctypes.c_void_p * 2)(*[t.data_ptr() for t in k])
    vp = (ctypes.c_void_p * 2)(*[t.data_ptr() for t in v])
    s, d = ints(src), ints(dst)
    _lib.check("pa_copy_blocks", _lib.call("pa_copy_blocks", kp, vp, _lib.PA_DTYPE_F16, ptr(s), ptr(d),
                                           None, 5, 2, 2, 8, 4, 6, ptr(status), stream()))
    assert int(status) == _lib.PA_DEVERR_BLOCK_ID
    assert torch.equal(bits(pool), want)


def test_no_pairs_and_another_stream():
    pool = make_pool(2, 6, 4, 2, 8, torch.float16)
    before = bits(pool).clone()
    k, v = layers(pool)
    ops.copy_blocks(k, v, ints([]), ints([]), torch.empty(0))
    assert torch.equal(bits(pool), before)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.copy_blocks(k, v, ints([1]), ints([5]), torch.empty(0))
    side.synchronize()
    assert torch.equal(bits(pool), expected(before.view(torch.float16), [1], [5], None, 6))


def test_offsets_past_32_bits():
    # one layer's K of 2.4e9 elements: pages at both ends
    NB, BS, H, D = 9200, 16, 64, 256
    k = torch.empty((NB, BS, H, D), dtype=torch.float8_e4m3fn, device="cuda")
    v = torch.empty((NB, BS, H, D), dtype=torch.float8_e4m3fn, device="cuda")
    assert k.numel() > 2**31
    for t, base in ((k, 1), (v, 2)):
        bits(t)[NB - 1] = base
        bits(t)[0] = base + 2
        bits(t)[NB - 2] = 0
        bits(t)[1] = 0
    ops.copy_blocks([k], [v], ints([NB - 1, 0]), ints([1, NB - 2]), torch.empty(0))
    for t, base in ((k, 1), (v, 2)):
        assert bool((bits(t)[1] == base).all()) and bool((bits(t)[NB - 2] == base + 2).all())


@pytest.mark.parametrize("shape", [(1, 1), (5, 33), (256, 200), (0, 4)])
def test_remap(shape):
    NB = 50
    g = torch.Generator().manual_seed(3)
    bt = torch.randint(-3, NB + 3, shape, dtype=torch.int32, generator=g).cuda()
    to = torch.randperm(NB, generator=g).to(torch.int32).cuda()
    got = ops.remap_block_tables(bt, to)
    inside = (bt >= 0) & (bt < NB)
    want = torch.where(inside, to[bt.clamp(0, NB - 1).long()], bt)
    assert torch.equal(got, want)


def test_shim_refusals():
    pool = make_pool(2, 6, 4, 2, 8, torch.float16)
    k, v = layers(pool)
    with pytest.raises(RuntimeError, match="one K and one V"):
        ops.copy_blocks(k, v[:1], ints([0]), ints([1]), torch.empty(0))
    with pytest.raises(RuntimeError, match="must be \\[n\\]"):
        ops.copy_blocks(k, v, ints([0]), ints([1, 2]), torch.empty(0))
    with pytest.raises(RuntimeError, match="num_rows"):
        ops.copy_blocks(k, v, ints([0, 1]), ints([2, 3]), ints([1]))
    with pytest.raises(RuntimeError, match="contiguous and alike"):
        ops.copy_blocks([t.transpose(0, 1) for t in k], v, ints([0]), ints([1]), torch.empty(0))
    with pytest.raises(RuntimeError, match="num_blocks"):
        ops.remap_block_tables(ints([[0]]), ints([[0, 1]]))


@pytest.mark.parametrize("layered", [True, False])
def test_fork_extend_free_compact(layered):
    BS, L, H, D = 16, 3, 2, 32
    alloc = TorchBlockAllocator(KVConfig(BS, 64, "float16"), ModelConfig(n_layer=L, n_head=H, head_dim=D),
                                "cuda:0", layered=layered)
    rng = np.random.default_rng(5)

    def content(t):  # [L, 2, T, H, D] of an allocation
        ids = torch.tensor(t.block_ids, dtype=torch.long, device="cuda")
        return torch.stack([alloc.pool[i][:, ids].reshape(2, len(ids) * BS, H, D)[:, :t.num_tokens]
                            for i in range(L)])

    dropped = alloc.allocate(range(20 * BS))
    a = alloc.allocate(range(37))
    k = rng.standard_normal((L, H, 37, D), dtype=np.float32)
    alloc.write_kv(a.block_ids, 0, k, -k)
    whole = content(a).clone()
    forks = alloc.fork(a, 3) + alloc.fork(a, 2, num_tokens=32) + alloc.fork(a, 1, num_tokens=0)
    assert [f.num_tokens for f in forks] == [37, 37, 37, 32, 32, 0]
    assert alloc.num_free_blocks == 64 - 20 - 3 - 3
    assert alloc.holders(a.block_ids[0]) == 6 and alloc.holders(a.block_ids[2]) == 1
    for f in forks[:3]:
        assert f.block_ids[:2] == a.block_ids[:2] and f.block_ids[2] not in a.block_ids
        assert torch.equal(content(f), whole)
    # forks grow apart; the parent stays
    for i, f in enumerate(forks[:3]):
        alloc.extend(f, range(20))
        assert len(f.block_ids) == 4
        kk = np.full((L, H, 20, D), float(i + 1), np.float32)
        alloc.write_kv(f.block_ids, 37, kk, kk)
    assert torch.equal(content(a), whole)
    grown = [content(f).clone() for f in forks]
    for i in range(3):
        assert torch.equal(grown[i][:, :, :37], whole) and bool((grown[i][:, :, 37:] == i + 1).all())
    # the parent ends, then a third of the pool; compaction keeps every content
    alloc.free(a.block_ids)
    assert alloc.holders(forks[0].block_ids[0]) == 5
    alloc.free(dropped.block_ids)
    table = alloc.block_table(forks)
    with pytest.raises(ValueError, match="no allocation"):
        alloc.compact(forks[1:3])
    block_map = alloc.compact(forks)
    used = 64 - alloc.num_free_blocks
    assert used == len({b for f in forks for b in f.block_ids})
    assert all(b < used for f in forks for b in f.block_ids)
    for f, want in zip(forks, grown):
        assert torch.equal(content(f), want)
    moved = ops.remap_block_tables(table, block_map)
    for i, f in enumerate(forks):
        assert moved[i, :len(f.block_ids)].tolist() == f.block_ids
    assert alloc.compact(forks) is None
    for f in forks:
        alloc.free(f.block_ids)
    assert alloc.num_free_blocks == 64 and sorted(alloc._free) == list(range(64)) and not alloc._shared


def test_fork_without_room_changes_nothing():
    alloc = TorchBlockAllocator(KVConfig(4, 3, "float16"), ModelConfig(n_layer=1, n_head=1, head_dim=32), "cuda:0")
    a = alloc.allocate(range(6))
    with pytest.raises(MemoryError):
        alloc.fork(a, 2)
    assert alloc.num_free_blocks == 1 and not alloc._shared
    with pytest.raises(ValueError):
        alloc.fork(a, 1, num_tokens=7)
    with pytest.raises(MemoryError):
        alloc.extend(a, range(20))
    assert a.num_tokens == 6
