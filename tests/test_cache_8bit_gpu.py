"""The 8-bit cache and the operators that write it, where a row has no place or no number."""
from __future__ import annotations

import math

import pytest
import torch

from nkilab import ops
from test_rotary_gpu import BF, DEV, F32, Cache8, freqs_of, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,block,dtype", [(16, 8, BF), (16, 4, F32), (64, 64, F32)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_no_append_writes_the_code_of_nan(page, block, dtype, value):
    """A block that gets a number that is none has the power NaN; its numbers are numbers."""
    T = 40
    x = torch.randn(1, 1, T, 2, 64, device=DEV).to(dtype)
    x[0, 0, 3, 0, 5] = x[0, 0, 3, 1] = x[0, 0, 39, 1, 63] = value
    for rotated in (False, True):
        c = Cache8(1, 6, 2, page, 64, block)
        for t in c.all:
            t.zero_()
        tables = i32([[5, 1, 3]])
        if rotated:
            ops.rotary_append(x[0], x[0], x[0], c.k[0], c.v[0], tables, i32([2]), freqs_of(64), None, k_scales=c.ks[0], v_scales=c.vs[0])
        else:
            ops.cache_append(x, x, c.k, c.v, tables, i32([2]), None, None, c.ks, c.vs)
        assert ((c.all[0] & 0x7f) != 0x7f).all()
        for s in (c.ks, c.vs):
            nan = s[0, tables[0].long()].transpose(0, 1).flatten(1).float().isnan()
            want = torch.zeros_like(nan)
            want[:, 5 // block] = want[1, 41 // block] = True
            assert torch.equal(nan, want)
