"""What paged_attention_shared refuses that a division must not meet."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PKG = Path(__file__).resolve().parents[1] / "gb10-attn_b200"


def test_a_pool_without_heads():
    """In a process of its own: a division by zero would end it."""
    code = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from pa_b200 import ops
ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
pool = torch.empty((4, 16, 0, 64), dtype=torch.float16, device="cuda")
q = torch.zeros((2, 8, 64), dtype=torch.float16, device="cuda")
try:
    ops.paged_attention_shared(q, pool, pool, ints([0], [1]), ints(3, 3), ints(0, 2), ints(2), 0.1)
except RuntimeError as e:
    print("refused:", e)
"""
    r = subprocess.run([sys.executable, "-c", code, str(PKG)], capture_output=True, text=True, timeout=200)
    assert r.returncode == 0 and "refused: n_head must be divisible" in r.stdout, (r.returncode, r.stdout, r.stderr[-400:])
