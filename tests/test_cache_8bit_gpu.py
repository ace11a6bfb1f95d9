"""The 8-bit cache and the operators that write it, where a row has no place or no number."""
from __future__ import annotations

import math

import pytest
import torch

from nkilab import ops
from test_rotary_gpu import BF, DEV, F32, Cache8, check, freqs_of, i32, turned

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


@pytest.mark.parametrize("dtype", [BF, F32])
def test_lengths_past_the_tables(dtype):
    """Rows behind the last page go nowhere, but count, and a token's position is its sequence's length and its place."""
    T, page, M = 3, 16, 2
    lens = [31, 32, 33, 70, 1 << 20, (1 << 30) + 5, -4]
    B = len(lens)
    tables = torch.arange(B * M, device=DEV).view(B, M).int()
    rows = torch.randn(1, B, T, 2, 64, device=DEV).to(dtype)
    c = Cache8(1, B * M, 2, page, 64, 8)
    plain = [torch.zeros(1, B * M, 2, page, 64, dtype=dtype, device=DEV) for _ in range(2)]
    want = ops.cache_append(rows, rows, *plain, tables, i32(lens), None, i32([T, T, T, T, T, T, 2]))
    was = c.bytes()
    got = ops.cache_append(rows, rows, c.k, c.v, tables, i32(lens), None, i32([T, T, T, T, T, T, 2]), c.ks, c.vs)
    assert got.tolist() == want.tolist() == [max(n, 0) + (2 if n < 0 else T) for n in lens]
    for b in range(1, B - 1):  # no row of these has a place
        for x, y in zip(c.all, was):
            assert torch.equal(x[:, :, b * M:(b + 1) * M], y[:, :, b * M:(b + 1) * M])
    f = freqs_of(64)
    q = torch.randn(B, T, 4, 64, device=DEV).to(dtype)
    at = i32([max(n, 0) for n in lens])[:, None] + torch.arange(T, device=DEV)
    for caches in ((c.k[0], c.v[0], c.ks[0], c.vs[0]), (plain[0][0], plain[1][0], None, None)):
        q2, k2 = ops.rotary_append(q, rows[0], rows[0], *caches[:2], tables, i32(lens), f, k_scales=caches[2], v_scales=caches[3])
        check(q2, *turned(q, at, f, False), dtype)
        check(k2, *turned(rows[0], at, f, False), dtype)
    now = c.bytes()
    for b in range(1, B - 1):
        for x, y in zip(now, was):
            assert torch.equal(x[:, :, b * M:(b + 1) * M], y[:, :, b * M:(b + 1) * M])
