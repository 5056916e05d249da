"""The example end to end, the allocator's batch helpers, and the steps under
graph capture."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

from pa_b200 import ops  # noqa: E402
from pa_b200.kv import Allocation, KVConfig, ModelConfig, TorchBlockAllocator  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(samples=8, prompt_len=203, steps=20), dict(samples=1, prompt_len=5, steps=4),
                                dict(samples=5, prompt_len=64, steps=6, heads=12, kv_heads=12, head_dim=64)])
def test_example_agrees_with_the_plain_decode(kw):
    """bf16 outputs: rounding of the weights and of the output, each 2^-8 of the largest at most."""
    from parallel_sampling import run
    r = run(check=True, **kw)
    assert r["worst"] <= 2 * 2.0 ** -8
    assert all(len(t) == kw["steps"] for t in r["text"])
    alloc, batch = r["alloc"], r["batch"]
    for a in batch:
        alloc.free(a.block_ids)
    assert alloc.num_free_blocks == alloc.kv_cfg.num_blocks and not alloc._shared


def test_prefix_groups():
    alloc = TorchBlockAllocator(KVConfig(4, 8, "float16"), ModelConfig(n_layer=1, n_head=1, head_dim=32), "cuda:0")

    def batch(*chains):
        return [Allocation(list(ids), n) for ids, n in chains]

    def groups(*chains):
        s, n = alloc.prefix_groups(batch(*chains))
        assert s.dtype == n.dtype == torch.int32 and s.is_cuda
        return s.tolist(), n.tolist()

    assert groups() == ([0], [])
    assert groups(([1, 2], 7)) == ([0, 1], [7])
    assert groups(([1, 2, 3], 10), ([1, 2, 4], 12), ([1, 2], 8)) == ([0, 3], [8])
    assert groups(([1, 2, 3], 10), ([1, 5], 6), ([6], 2), ([1, 2], 8)) == ([0, 2, 3, 4], [4, 2, 8])
    assert groups(([], 0), ([], 0), ([1], 3), ([1], 2)) == ([0, 1, 2, 4], [0, 0, 2])


def test_graph_capture_follows_new_lengths():
    """One captured step, replayed with other positions, lengths and values in the same buffers."""
    B, H, HKV, D = 6, 8, 2, 64
    cfg = ModelConfig(n_layer=1, n_head=H, head_dim=D, n_kv_head=HKV)
    alloc = TorchBlockAllocator(KVConfig(16, 64, "bfloat16"), cfg, "cuda:0")
    parent = alloc.allocate(range(100))
    g = torch.Generator(device="cuda").manual_seed(0)
    k0 = torch.randn((1, HKV, 100, D), device="cuda", generator=g)
    alloc.write_kv(parent.block_ids, 0, k0, -k0)
    batch = alloc.fork(parent, B)
    for a in batch:
        alloc.extend(a, range(20))
    table, (starts, lens) = alloc.block_table(batch), alloc.prefix_groups(batch)
    cos_sin = ops.rope_table(128, D)
    qkv = torch.randn((B, H + 2 * HKV, D), device="cuda", generator=g).bfloat16()
    pos = torch.full((B,), 100, dtype=torch.int32, device="cuda")
    ctx = pos + 1

    def step():
        return alloc.layer_step_shared(0, *qkv.split((H, HKV, HKV), 1), None, None, cos_sin, pos, table, ctx, starts,
                                       lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(4):
        qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=g))
        pos.fill_(100 + n)
        ctx.fill_(101 + n)
        ctx[n] = pos[n] = 0 if n == 3 else 101 + n
        pos[n] = -1 if n == 3 else 100 + n
        graph.replay()
        got = out.clone()
        torch.testing.assert_close(got, step(), rtol=0, atol=0, equal_nan=True)
        assert bool(got[3].isnan().all()) == (n == 3)
