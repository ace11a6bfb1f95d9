"""What the sines, the scales' layout and the rounding of an 8-bit cache have to hold to, closer than the operators' own
tests say it."""
from __future__ import annotations

import math

import pytest
import torch

from nkilab import ops
from nkilab.serving import PagedCache, Rotary, decode, extend
from test_rotary_gpu import BF, DEV, E4M3, F32, Cache8, freqs_of, i32
from test_serving_step_gpu import blocks_of, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("magnitude", [1.0, 1.25])
def test_sines_and_cosines_are_rounded_once(interleaved, magnitude):
    """Pairs (1, 0) and (0, 1) come out as (c, s) and (-s, c): the products with 0 and 1 and their sums are exact, so that
    what is left is half a step, 2^-24 of the number, and what the angle's reduction in 64 bits leaves: three roundings of
    2^-53 of up to 2^20 radians (3.5e-10), and the series' 7e-12. In 32 bits the angle alone would be off by up to 9e-8."""
    T, d = 4099, 128
    f = freqs_of(d)
    at = torch.randint(0, 1 << 20, (2, T), dtype=torch.int32, device=DEV)
    pair = torch.tensor([[1.0, 0.0], [0.0, 1.0]], device=DEV)  # of the two heads
    x = torch.empty(2, T, 2, d, device=DEV)
    if interleaved:
        x.view(2, T, 2, d // 2, 2)[:] = pair[:, None]
    else:
        x.view(2, T, 2, 2, d // 2)[:] = pair[:, :, None]
    y = ops.rotary(x, at, f, None, interleaved, magnitude).double()
    y = y.unflatten(-1, (d // 2, 2)) if interleaved else y.unflatten(-1, (2, d // 2)).transpose(-1, -2)
    angle = at.double()[..., None] * f
    c, s = angle.cos() * magnitude, angle.sin() * magnitude
    want = torch.stack([torch.stack([c, s], -1), torch.stack([-s, c], -1)], 2)
    assert ((y - want).abs() <= 2.0 ** -24 * want.abs() + 5e-10 * magnitude).all()


def test_scales_that_are_not_contiguous_are_refused():
    c, tables, lens = Cache8(1, 4, 2, 32, 64, 16), i32([[0], [1]]), i32([3, 4])
    rows = torch.randn(2, 3, 2, 64, device=DEV).to(BF)
    turned = c.ks[0].mT.contiguous().mT
    assert turned.shape == c.ks[0].shape and not turned.is_contiguous()
    was = c.bytes()
    for ks, vs in ((turned, c.vs[0]), (c.ks[0], turned)):
        for call in (lambda: ops.rotary_append(rows, rows, rows, c.k[0], c.v[0], tables, lens, freqs_of(64), k_scales=ks, v_scales=vs),
                     lambda: ops.cache_append(rows, rows, c.k[0], c.v[0], tables, lens, None, None, ks, vs),
                     lambda: ops.attention_tree(rows, rows, rows, c.k[0], c.v[0], tables, lens, None, None, ks, vs)):
            with pytest.raises(RuntimeError, match="contiguous"):
                call()
    for x, y in zip(c.all, was):
        assert torch.equal(x, y)


@pytest.mark.parametrize("block", [4, 16])
def test_one_pass_and_two_differ_by_a_rounding_to_bf16(block):
    """extend rounds turned keys once, from 32 bits to e4m3, decode and append twice. Each number is within half a step of
    its grid, 2^-4 of it or 2^-10 of its scale, of values that are within bf16's 2^-8 of each other."""
    blocks, rotary = blocks_of(2), Rotary(64)
    a, b = (PagedCache(2, 2, 30, 4, 64, page_size=16, dtype=E4M3, block=block) for _ in range(2))
    x = torch.randn(2, 100, 256, device=DEV).to(BF)
    for c in (a, b):
        c.reserve(100)
    extend(blocks, x, a, rotary)
    _, k, v = decode(blocks, x, b, None, rotary)
    b.append(k, v)
    for slot in range(2):
        got, want = values(a, slot), values(b, slot)
        assert torch.equal(got[1], want[1])
        tables = [c.tables[slot, :7].long() for c in (a, b)]
        steps = [c.k_scales[:, t].float().repeat_interleave(block, -1).transpose(1, 2).flatten(2, 3)[:, :, :100, None] for c, t in zip((a, b), tables)]
        p, q = got[0].double(), want[0].double()
        # x with |p - x| <= 2^-4 |p| (1 + 2^-4) + .., so in numbers of the grids themselves a little more than half a step
        bound = (2.0 ** -4 / (1 - 2.0 ** -4)) * (p.abs() + q.abs()) + 1.1 * 2.0 ** -8 * torch.maximum(p.abs(), q.abs()) + 2.0 ** -10 * (steps[0] + steps[1]).double()
        assert ((p - q).abs() <= bound).all()
        # and most are the same numbers: a second rounding moves those within 2^-8 of a border between two, steps being 2^-3 or so
        assert (p != q).double().mean() < 0.15
