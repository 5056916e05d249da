"""The allocator's counted holds, on the host alone: forks at a page's end copy nothing."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from pa_b200.kv import KVConfig, ModelConfig, TorchBlockAllocator


def make(blocks=16):
    return TorchBlockAllocator(KVConfig(4, blocks, "float16"), ModelConfig(n_layer=1, n_head=1, head_dim=32), "cpu")


@pytest.mark.parametrize("form", [list, tuple, iter, np.asarray, torch.tensor])
def test_a_hold_is_given_up_whatever_form_the_ids_come_in(form):
    alloc = make()
    a = alloc.allocate(range(12))
    fork, = alloc.fork(a)
    assert fork.block_ids == a.block_ids and alloc.num_free_blocks == 13
    alloc.free(form(a.block_ids))
    assert alloc.num_free_blocks == 13 and all(alloc.holders(b) == 1 for b in fork.block_ids)
    alloc.free(form(fork.block_ids))
    assert sorted(alloc._free) == list(range(16)) and all(type(b) is int for b in alloc._free) and not alloc._shared
    again = alloc.allocate(range(64))
    assert sorted(again.block_ids) == list(range(16))
