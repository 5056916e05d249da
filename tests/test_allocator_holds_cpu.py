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


def test_a_fork_whose_copy_fails_changes_nothing(monkeypatch):
    alloc = make()
    a = alloc.allocate(range(10))
    free = list(alloc._free)

    def fail(*_):
        raise RuntimeError("no copy")

    monkeypatch.setattr(alloc, "copy_blocks", fail)
    with pytest.raises(RuntimeError, match="no copy"):
        alloc.fork(a, 3)
    assert alloc._free == free and not alloc._shared
    monkeypatch.setattr(alloc, "copy_blocks", lambda *_: None)
    forks = alloc.fork(a, 3)
    assert alloc.holders(a.block_ids[0]) == 4 and alloc.holders(a.block_ids[2]) == 1
    assert len({f.block_ids[2] for f in forks} | {a.block_ids[2]}) == 4
