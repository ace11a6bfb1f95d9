"""Calls of nkilab.serving that bring no token."""
from __future__ import annotations

import pytest
import torch

from nkilab.serving import PagedCache, Rotary, decode, extend
from test_serving_step_gpu import BF, DEV, E4M3, F32, blocks_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32, E4M3])
def test_no_new_tokens(dtype):
    blocks, rotary, rows = blocks_of(2), Rotary(64), F32 if dtype == F32 else BF
    cache = PagedCache(2, 2, 8, 4, 64, page_size=16, dtype=dtype)
    cache.reserve(20)
    x = torch.randn(2, 9, 256, device=DEV).to(rows)
    extend(blocks, x, cache, rotary)
    was = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.tables, cache.lens)]
    for count in (None, torch.tensor([0, 3], dtype=torch.int32, device=DEV)):
        y = extend(blocks, x[:, :0], cache, rotary, count)
        assert y.shape == (2, 0, 256) and y.dtype == rows and y.device == x.device
    y, k, v = decode(blocks, x[:, :0], cache, None, rotary)
    assert y.shape == (2, 0, 256) and k.shape == v.shape == (2, 2, 0, 4, 64)
    for now, t in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.tables, cache.lens), was):
        assert torch.equal(now, t)
