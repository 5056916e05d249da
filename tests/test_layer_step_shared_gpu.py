"""TorchBlockAllocator.layer_step_shared: what it refuses, it refuses before it writes to the pool."""
from __future__ import annotations

import pytest
import torch

from pa_b200 import ops
from pa_b200.kv import KVConfig, ModelConfig, TorchBlockAllocator

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pool,source,change,text", [
    ("float8_e4m3fn", torch.float16, {}, "float16"),
    ("float32", torch.float32, {}, "float16"),
    ("bfloat16", torch.float32, {}, "float16"),
    ("bfloat16", torch.float16, {}, "float16"),
    ("float16", torch.float16, {"heads": 7}, "multiple|divisible"),
    ("float16", torch.float16, {"starts": [0]}, "group_starts"),
    ("float16", torch.float16, {"ctx": [21]}, "context_lens"),
])
def test_refusals_leave_the_pool_alone(pool, source, change, text):
    heads = change.get("heads", 8)
    alloc = TorchBlockAllocator(KVConfig(16, 8, pool), ModelConfig(n_layer=1, n_head=8, head_dim=64, n_kv_head=2),
                                "cuda:0")
    batch = alloc.fork(alloc.allocate(range(20)), 2)
    for a in batch:
        alloc.extend(a, [0])
    table, (starts, lens) = alloc.block_table(batch), alloc.prefix_groups(batch)
    if "starts" in change:
        starts = torch.tensor(change["starts"], dtype=torch.int32, device="cuda")
    ctx = torch.tensor(change.get("ctx", [21, 21]), dtype=torch.int32, device="cuda")
    q, k, v = torch.ones((2, heads + 4, 64), device="cuda").to(source).split((heads, 2, 2), 1)
    pos = torch.tensor([20, 20], dtype=torch.int32, device="cuda")
    with pytest.raises((ValueError, RuntimeError), match=text):
        alloc.layer_step_shared(0, q, k, v, None, None, ops.rope_table(32, 64), pos, table, ctx, starts, lens)
    for x in alloc.layer_kv(0):
        assert not bool(x.float().any())
