"""Calls that are the first of their process, before a larger one has asked for more shared memory."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

from conftest import PKG

pytestmark = pytest.mark.gpu

APPENDS = """
import torch
from nkilab import ops
for d, block, dtype in ((96, 16, torch.bfloat16), (64, 24, torch.bfloat16), (48, 32, torch.bfloat16), (96, 8, torch.float32), (48, 16, torch.float32)):
    k, v = (torch.zeros(1, 4, 2, 96, d, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(1, 4, 2, 96 // block, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2))
    rows, tables, lens = torch.ones(1, 1, 5, 2, d, device="cuda", dtype=dtype), torch.tensor([[2]], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda")
    assert ops.cache_append(rows, rows, k, v, tables, lens, None, None, ks, vs).tolist() == [8]
    assert (k[0, 2, :, 3:8].float() * ks[0, 2, :, :1, None].float() == 1).all()
"""


def test_appends_whose_rows_take_48_kilobytes():
    """The two buffers of each of eight warps are 48 KB exactly, with rows of 96 in blocks of 16 for instance."""
    out = subprocess.run([sys.executable, "-c", APPENDS], env=dict(os.environ, PYTHONPATH=PKG), capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
