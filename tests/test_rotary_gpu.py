"""Rotary positions and appends with the rotation on the way, against plain statements of them in
64 bits, at the sizes and values where they can go wrong."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nkilab import _native as N
from nkilab import ops

pytestmark = pytest.mark.gpu

BF, F32, E4M3, E8M0 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float8_e8m0fnu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def freqs_of(part, base=10000.0):
    return ops.rotary_frequencies(part, base)[0]


def turned(x, positions, freqs, interleaved, magnitude=1.0):
    """(the formula's result, |x1| + |x2| of each entry's pair) in 64 bits, on the CPU."""
    x, f = x.detach().double().cpu(), freqs.cpu()
    n = f.numel()
    y, mag = x.clone(), x.abs()
    angle = positions.cpu().double()[..., None, None] * f
    c, s = angle.cos(), angle.sin()
    i = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    j = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = (a * c - b * s) * magnitude, (b * c + a * s) * magnitude
    mag[..., i] = mag[..., j] = (a.abs() + b.abs()) * magnitude
    return y, mag


def check(got, want, mag, dtype):
    """A sine or cosine: the angle as a part of a turn, doubled, is rounded to 32 bits (pi 2^-25) and the
    function is off by up to two steps (2^-23); products and sum round three times: together
    under 6e-7 of |x1| + |x2|. In bf16 the result's rounding, half a step, besides."""
    bound = 6e-7 * mag + (2.0 ** -8 * want.abs() if dtype == BF else 0) + 1e-38
    err = (got.detach().double().cpu() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())


def depths(parents):
    """As in the attention: a child of an absent or not earlier token is one of the last cached position."""
    out = []
    for row in parents:
        d = []
        for i, p in enumerate(row):
            n, at = 0, i
            while 0 <= row[at] < at and row[row[at]] >= -1 and row[i] >= -1:
                at = row[at]
                n += 1
            d.append(n)
        out.append(d)
    return out


SHAPES = [
    # B, T, H, d, part, dtype
    (1, 1, 40, 128, 128, BF),
    (1, 1, 1, 8, 8, BF),
    (2, 3, 5, 64, 64, F32),
    (3, 7, 12, 80, 40, BF),        # pairs 20 entries apart: half vectors
    (2, 5, 3, 80, 40, F32),
    (1, 33, 2, 128, 16, BF),
    (4, 2, 7, 24, 8, F32),
    (2, 9, 6, 256, 256, F32),
    (1, 4, 3, 256, 8, BF),
    (64, 1, 9, 96, 96, BF),
    (1, 1300, 3, 128, 64, BF),     # groups of 2 tokens
    (2, 2501, 1, 64, 64, F32),     # of 8, the last one short
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,d,part,dtype", SHAPES)
def test_rotary(B, T, H, d, part, dtype, interleaved):
    g = torch.Generator(device=DEV).manual_seed(d + T)
    x = torch.randn(B, T, H + 2, d, generator=g, device=DEV).to(dtype)[:, :, :H]
    f = freqs_of(part)
    start = torch.randint(0, 1 << 20, (B,), generator=g, device=DEV).int()
    each = torch.randint(-5, 1 << 30, (B, T), generator=g, device=DEV).int()
    got = ops.rotary(x, start, f, interleaved=interleaved)
    assert got.is_contiguous() and got.dtype == dtype
    check(got, *turned(x, start[:, None] + torch.arange(T, device=DEV), f, interleaved), dtype)
    check(ops.rotary(x, each, f, interleaved=interleaved, magnitude=1.25), *turned(x, each, f, interleaved, 1.25), dtype)


def test_rotary_equals_rope():
    """The older operator's case: whole heads, the half layout, one offset."""
    x = torch.randn(5, 40, 64, device=DEV)
    want = ops.rope(x, 10000.0, 7)
    got = ops.rotary(x.transpose(0, 1)[None], i32([7]), freqs_of(64))[0].transpose(0, 1)
    # rope's angle is rounded to 32 bits: 46 radians times 2^-23
    assert (got - want).abs().max() < 2e-5


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotary_trees(dtype):
    r = np.random.RandomState(3)
    for B, T in ((1, 1), (3, 40), (2, 128)):
        parents = [[-2 if r.rand() < 0.2 else r.randint(-1, max(i, 1)) if i else -1 for i in range(T)] for _ in range(B)]
        parents[0] = list(range(-1, T - 1))
        if T > 3:
            parents[-1][3], parents[-1][1] = 3, T - 1  # itself, a later one
        x = torch.randn(B, T, 4, 64, device=DEV).to(dtype)
        start = i32(r.randint(0, 70000, B).tolist())
        f = freqs_of(64)
        at = start.cpu()[:, None] + torch.tensor(depths(parents))
        got = ops.rotary(x, start, f, i32(parents))
        check(got, *turned(x, at, f, False), dtype)
        assert torch.equal(got[0], ops.rotary(x, start, f)[0])  # a chain


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotary_gradient(dtype, interleaved):
    B, T, H, d, part = 2, 11, 3, 80, 48
    x = torch.randn(B, T, H, d, device=DEV).to(dtype).requires_grad_()
    g = torch.randn(B, T, H, d, device=DEV).to(dtype)
    f, at = freqs_of(part), i32([[5 * b + 3 * t for t in range(T)] for b in range(B)])
    y = ops.rotary(x, at, f, interleaved=interleaved, magnitude=1.5)
    y.backward(g)
    want, mag = turned(g, -at, f, interleaved, 1.5)
    check(x.grad, want, mag, dtype)
    if dtype == F32:
        # differences: the sum of y g is linear in x, so that they are off by roundings alone
        # (of some 5000 products, each below 40, times 2^-24, over the step)
        for b, t, h, e in ((0, 0, 0, 0), (1, 10, 2, 47), (1, 5, 1, 24), (0, 3, 2, 79)):
            parts = []
            for step in (0.5, -0.5):
                z = x.detach().clone()
                z[b, t, h, e] += step
                parts.append((ops.rotary(z, at, f, interleaved=interleaved, magnitude=1.5).double() * g.double()).sum())
            assert abs(parts[0] - parts[1] - x.grad[b, t, h, e].double()) < 2e-5
        # the gradient's own gradient is the operator again
        (dx,) = torch.autograd.grad(ops.rotary(x, at, f, interleaved=interleaved, magnitude=1.5), x, g.requires_grad_(), create_graph=True)
        (dg,) = torch.autograd.grad(dx, g, torch.ones_like(g))
        check(dg, *turned(torch.ones_like(g), at, f, interleaved, 1.5), dtype)
    # an expanded gradient, and none needed
    x.grad = None
    ops.rotary(x, at, f, interleaved=interleaved).sum().backward()
    check(x.grad, *turned(torch.ones(B, T, H, d), -at, f, interleaved), dtype)
    with torch.no_grad():
        assert not ops.rotary(x, at, f).requires_grad


def test_rotary_layouts():
    f, at = freqs_of(64), i32([3, 70])
    base = torch.randn(2, 6, 5, 64, device=DEV).to(BF)
    want = ops.rotary(base, at, f)
    wide = torch.zeros(2, 6, 5, 72, device=DEV, dtype=BF)
    wide[..., :64] = base
    assert torch.equal(ops.rotary(wide[..., :64], at, f), want)
    assert torch.equal(ops.rotary(base.transpose(1, 2).contiguous().transpose(1, 2), at, f), want)
    odd = torch.zeros(base.numel() + 1, device=DEV, dtype=BF)[1:].view_as(base).copy_(base)  # off a 16-byte boundary
    assert torch.equal(ops.rotary(odd, at, f), want)
    assert torch.equal(ops.rotary(base[..., ::1].mT.contiguous().mT, at, f), want)
    one = base[:1, :1].expand(2, 6, 5, 64)
    assert torch.equal(ops.rotary(one, at, f), ops.rotary(one.contiguous(), at, f))
    assert ops.rotary(base[:0], at[:0], f).shape == (0, 6, 5, 64)
    assert ops.rotary(base[:, :0], at, f).shape == (2, 0, 5, 64)
    special = base.clone()
    special[0, 0, 0, 0], special[0, 1, 0, 0], special[1, 0, 0, 40] = float("nan"), float("inf"), float("-inf")
    assert torch.equal(ops.rotary(special, at, f).isfinite(), turned(special, at[:, None] + torch.arange(6, device=DEV), f, False)[0].isfinite().to(DEV))


def test_rotary_streams_and_graphs():
    x, f = torch.randn(3, 17, 8, 128, device=DEV).to(BF), freqs_of(128)
    at = i32([1, 2, 3])
    want = ops.rotary(x, at, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.rotary(x, at, f), want)
        leaf = x.clone().requires_grad_()
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            y = ops.rotary(leaf, at, f)
            (dx,) = torch.autograd.grad(y, leaf, x)
    at.add_(9)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ops.rotary(x, at, f))
    again = x.clone().requires_grad_()
    assert torch.equal(dx, torch.autograd.grad(ops.rotary(again, at, f), again, x)[0])


def test_rotary_past_32_bits():
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    x = torch.empty(2, 1 << 16, 130, 128, device=DEV, dtype=BF)  # 2.2e9 elements
    x[1, -4:].normal_()
    f = freqs_of(128)
    got = ops.rotary(x, i32([0, 100]), f)
    assert torch.equal(got[1, -4:], ops.rotary(x[1:, -4:], i32([100 + (1 << 16) - 4]), f)[0])


# --------------------------------------------------------------------------- appends

def power(top):
    """The smallest e >= -100 with top <= 448 2^e."""
    if top == 0:
        return -100
    e = int(np.floor(np.log2(top / 448)))
    while 448 * 2.0 ** e < top:
        e += 1
    while 448 * 2.0 ** (e - 1) >= top:
        e -= 1
    return max(e, -100)


def e4m3(x):
    """Ties to even; the codes of values up to 448."""
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -20))), -6)
    return np.round(x * 2.0 ** (3 - e)) * 2.0 ** (e - 3)


class Reference:
    """A slot's rows of one (layer, head) of k or v in 8 bits, in 64 bits on the host."""

    def __init__(self, block):
        self.block, self.rows, self.powers = block, [], []

    def extend(self, rows):
        """Whole blocks at a time: what one call brings is in its block's power together."""
        at = 0
        while at < len(rows):
            n, first = len(self.rows), len(self.rows) // self.block * self.block
            new = rows[at:at + self.block - n % self.block]
            top = np.abs(new).max() if new.size else 0.0
            e = power(top) if np.isfinite(top) else None
            if n > first:
                was = self.powers[-1]
                e = None if was is None or e is None else max(e, was)
                if e is not None and e > was:
                    for i in range(first, n):
                        self.rows[i] = e4m3(self.rows[i] * 2.0 ** (was - e))
                self.powers[-1] = e
            else:
                self.powers.append(e)
            self.rows += list(e4m3(new * 2.0 ** -e) if e is not None else new * np.nan)
            at += len(new)


class Cache8:
    def __init__(self, L, P, Hkv, page, d, block, strided=False):
        junk = torch.randint(0, 255, (2, L, P, page, Hkv, d) if strided else (2, L, P, Hkv, page, d), device=DEV).to(torch.uint8)
        kv = junk.view(E4M3).transpose(3, 4) if strided else junk.view(E4M3)
        self.k, self.v = kv
        scales = torch.randint(0, 255, (2, L, P, Hkv, page // block), device=DEV).to(torch.uint8)
        self.ks, self.vs = scales.view(E8M0)
        self.all = (junk, scales)

    def bytes(self):
        return [t.clone() for t in self.all]


APPEND8 = [
    # L, Hkv, page, d, block, dtype, calls: (lens are kept, rows of each slot)
    (1, 2, 16, 64, 16, BF, [[1, 5], [1, 1], [14, 0], [1, 12]]),
    (2, 3, 64, 128, 16, F32, [[7, 0, 16], [1, 1, 1], [40, 33, 2]]),
    (1, 8, 24, 80, 8, BF, [[10, 3], [1, 30]]),
    (3, 1, 32, 16, 4, BF, [[1, 2], [3, 3], [6, 9]]),
    (1, 2, 8, 128, 1, F32, [[3, 4], [1, 9]]),
    (1, 2, 24, 112, 24, BF, [[23, 1], [2, 23], [30, 24]]),
    (1, 4, 128, 64, 128, BF, [[100, 1], [29, 127], [3, 1]]),
    (1, 2, 256, 128, 256, F32, [[300, 200], [1, 60]]),
    (2, 5, 64, 128, 32, F32, [[33, 31], [64, 1]]),
]


@pytest.mark.parametrize("grow", [0.0, 2.0, -2.0])
@pytest.mark.parametrize("at", range(len(APPEND8)))
def test_append_8bit(at, grow):
    """Codes and powers bit for bit; bytes of rows that no call writes stay."""
    L, Hkv, page, d, block, dtype, calls = APPEND8[at]
    B = len(calls[0])
    r = np.random.RandomState(at)
    M = -(-max(sum(c[b] for c in calls) for b in range(B)) // page) + 1
    P = B * M + 2
    cache = Cache8(L, P, Hkv, page, d, block, strided=at % 2 == 1)
    tables = i32(r.permutation(P)[:B * M].reshape(B, M).tolist())
    lens = i32([0] * B)
    want = {(l, b, h, c): Reference(block) for l in range(L) for b in range(B) for h in range(Hkv) for c in "kv"}
    scale = 1.0
    before = cache.bytes()
    for n in calls:
        T = max(n) + 2
        rows = [(torch.randn(L, B, T, Hkv, d, device=DEV) * scale * 2.0 ** torch.randint(-4, 4, (L, B, T, Hkv, 1), device=DEV)).to(dtype) for _ in range(2)]
        path = np.full((B, T), -1)
        for b in range(B):
            path[b, :n[b]] = np.sort(r.choice(T, n[b], replace=False))
        lens = ops.cache_append(*rows, cache.k, cache.v, tables, lens, i32(path.tolist()), i32(n), cache.ks, cache.vs)
        for (l, b, h, c), ref in want.items():
            ref.extend(rows["kv".index(c)][l, b, path[b, :n[b]], h].double().cpu().numpy())
        scale *= 2.0 ** grow
    assert lens.tolist() == [sum(c[b] for c in calls) for b in range(B)]
    written = [torch.zeros_like(t, dtype=torch.bool) for t in cache.all]
    for i, c in enumerate("kv"):
        codes, scales = (cache.k, cache.ks) if c == "k" else (cache.v, cache.vs)
        mark = written[0][i] if not at % 2 else written[0][i].transpose(2, 3)
        for l in range(L):
            for b in range(B):
                for h in range(Hkv):
                    ref = want[l, b, h, c]
                    for p in range(len(ref.rows)):
                        pg = int(tables[b, p // page])
                        mark[l, pg, h, p % page] = True
                        written[1][i][l, pg, h, p % page // block] = True
                    if ref.rows:
                        pages = tables[b, :-(-len(ref.rows) // page)].long()
                        got = codes[l, pages, h].reshape(-1, d)[:len(ref.rows)].double().cpu().numpy()
                        np.testing.assert_array_equal(got, np.stack(ref.rows))
                        exps = scales[l, pages, h].reshape(-1)[:len(ref.powers)].view(torch.uint8).cpu().tolist()
                        assert exps == [e + 127 for e in ref.powers]
    for now, was, mark in zip(cache.all, before, written):
        assert torch.equal(now[~mark], was[~mark])


def test_append_8bit_values():
    """Zeros, the smallest and largest magnitudes, the borders between powers, infinities and NaN."""
    d, block = 16, 4
    cache = Cache8(1, 8, 1, 16, d, block)
    rows = torch.zeros(1, 1, 32, 1, d, device=DEV)
    tops = [0.0, 448.0, np.nextafter(np.float32(448), np.float32(1e9)), 449.0, 1e-45, 2.0 ** -100, 3.4e38, 2.0 ** -92]
    for i, t in enumerate(tops):
        rows[0, 0, 4 * i, 0, 3] = -float(t)
        rows[0, 0, 4 * i + 2, 0, 5] = float(t) / 3
    tables = i32([[5, 2]])
    ops.cache_append(rows, rows, cache.k, cache.v, tables, i32([0]), None, None, cache.ks, cache.vs)
    ref = Reference(block)
    ref.extend(rows[0, 0, :, 0].double().cpu().numpy())
    assert cache.ks[0, [5, 2], 0].reshape(-1).view(torch.uint8).tolist() == [e + 127 for e in ref.powers]
    np.testing.assert_array_equal(cache.k[0, [5, 2], 0].reshape(-1, d).double().cpu().numpy(), np.stack(ref.rows))
    # not finite: the block's power is NaN, and stays so; its neighbours' are not
    rows = torch.ones(1, 1, 16, 1, d, device=DEV)
    rows[0, 0, 1, 0, 0], rows[0, 0, 9, 0, 15] = float("inf"), float("nan")
    lens = ops.cache_append(rows, torch.ones_like(rows), cache.k, cache.v, tables, i32([0]), None, i32([14]), cache.ks, cache.vs)
    assert cache.ks[0, 5, 0].float().isnan().tolist() == [True, False, True, False]
    assert not cache.vs[0, 5].float().isnan().any()
    ops.cache_append(torch.ones_like(rows), rows * float("-inf"), cache.k, cache.v, tables, lens, None, i32([1]), cache.ks, cache.vs)
    assert cache.ks[0, 5, 0].float().isnan().tolist() == [True, False, True, False]
    assert cache.vs[0, 5, 0].float().isnan().tolist() == [False, False, False, True]


ROTARY_APPEND = [
    # H, Hkv, page, d, part, block (0: the rows' type), dtype, interleaved, lens, T, count
    (8, 2, 16, 64, 64, 16, BF, False, [0, 5], 1, None),
    (4, 4, 64, 128, 128, 16, BF, False, [30, 0, 63], 37, [37, 20, 0]),
    (6, 3, 24, 80, 40, 8, BF, False, [11, 100], 19, None),
    (12, 4, 24, 64, 32, 0, BF, True, [500, 3], 31, [31, 7]),
    (2, 1, 32, 128, 128, 32, F32, True, [1, 31], 70, None),
    (3, 3, 128, 128, 64, 128, F32, False, [100, 0], 200, [200, 140]),
    (4, 2, 17, 96, 96, 0, F32, False, [16, 0], 18, None),
    (4, 2, 8, 16, 16, 2, BF, True, [3, 4], 6, [6, 0]),
    (2, 2, 64, 128, 128, 64, BF, True, [9], 130, None),
    (32, 32, 64, 128, 128, 16, BF, False, [0], 700, None),
]


@pytest.mark.parametrize("at", range(len(ROTARY_APPEND)))
def test_rotary_append(at):
    H, Hkv, page, d, part, block, dtype, interleaved, lens, T, count = ROTARY_APPEND[at]
    r, B = np.random.RandomState(at), len(lens)
    g = torch.Generator(device=DEV).manual_seed(at)
    M = -(-(max(lens) + T) // page) + 1
    P = B * M + 2
    tables = i32(r.permutation(P)[:B * M].reshape(B, M).tolist())
    qkv = torch.randn(B, T, H + 2 * Hkv, d, generator=g, device=DEV).to(dtype)
    q, k, v = qkv.split([H, Hkv, Hkv], 2)
    f, ln, ct = freqs_of(part), i32(lens), None if count is None else i32(count)
    want_q, want_k = (ops.rotary(t, ln, f, interleaved=interleaved, magnitude=1.1) for t in (q, k))
    counts = count or [T] * B
    if not block:
        caches = [torch.randn(P, Hkv, page, d, generator=g, device=DEV).to(dtype) for _ in range(2)]
        other = [c.clone() for c in caches]
        got_q, got_k = ops.rotary_append(q, k, v, *caches, tables, ln, f, ct, interleaved, 1.1)
        ops.cache_append(want_k[None], v[None], other[0][None], other[1][None], tables, ln, None, ct)
        assert torch.equal(caches[0], other[0]) and torch.equal(caches[1], other[1])
    else:
        a, b = Cache8(1, P, Hkv, page, d, block), Cache8(1, P, Hkv, page, d, block)
        a.all[1].clamp_(100, 140)  # what earlier rows left
        for x, y in zip(b.all, a.all):
            x.copy_(y)
        got_q, got_k = ops.rotary_append(q, k, v, a.k[0], a.v[0], tables, ln, f, ct, interleaved, 1.1, a.ks[0], a.vs[0])
        # the same rows, turned in 32 bits before: the operator rounds them once
        k32 = ops.rotary(k.float(), ln, f, interleaved=interleaved, magnitude=1.1)
        ops.cache_append(k32[None], v.float()[None], b.k, b.v, tables, ln, None, ct, b.ks, b.vs)
        for x, y in zip(a.all, b.all):
            assert torch.equal(x, y)
        exact, mag = turned(k, ln[:, None] + torch.arange(T, device=DEV), f, interleaved, 1.1)
        values = a.k[0].double().cpu().unflatten(2, (-1, block)) * a.ks[0].double().cpu()[..., None, None]
        step = a.ks[0].double().cpu()[..., None, None].expand(values.shape).flatten(2, 3) * 2.0 ** -10
        values = values.flatten(2, 3)
        for s in range(B):
            for j in range(counts[s]):
                p, slot = int(tables[s, (lens[s] + j) // page]), (lens[s] + j) % page
                err = (values[p, :, slot] - exact[s, j]).abs()
                assert (err <= 2.0 ** -4 * exact[s, j].abs() * 1.001 + step[p, :, slot] + 1e-6 * mag[s, j]).all()
    assert torch.equal(got_q, want_q) and torch.equal(got_k, want_k)


def test_rotary_append_drops_rows_without_a_page():
    tables = i32([[2, -1, 9], [0, 1, 3]])
    for bits8 in (False, True):
        c = Cache8(1, 4, 2, 8, 32, 8)
        c.all[1].fill_(140)  # more than the new rows need: the old ones stay as they are
        plain = [torch.zeros(4, 2, 8, 32, device=DEV, dtype=BF) for _ in range(2)]
        was = c.bytes()
        q, k, v = (torch.randn(2, 30, h, 32, device=DEV).to(BF) for h in (4, 2, 2))
        lens, f = i32([-3, 20]), freqs_of(32)
        if bits8:
            out = ops.rotary_append(q, k, v, c.k[0], c.v[0], tables, lens, f, None, False, 1.0, c.ks[0], c.vs[0])
            same = [x == y for x, y in zip(c.all, was)]
            assert same[0][:, 0, [0, 1]].all() and same[1][:, 0, [0, 1]].all()  # slot 1 is behind them
            assert same[0][:, 0, 3, :, :4].all() and not same[0][:, 0, 3, :, 4:].all() and not same[0][:, 0, 2].all()
            assert same[1][:, 0, 3].all() and not same[1][:, 0, 2].any()
        else:
            out = ops.rotary_append(q, k, v, *plain, tables, lens, f)
            assert not plain[0][[0, 1]].any() and not plain[0][3, :, :4].any() and plain[0][3, :, 4:].any() and plain[0][2].any()
        assert torch.equal(out[0], ops.rotary(q, lens.clamp_min(0), f))


def test_append_8bit_repeats_streams_and_graphs():
    """Equal calls give equal bytes, on another stream and from a graph; the second of two calls on
    the same rows changes nothing."""
    f, tables, lens = freqs_of(64), i32([[0, 1, 2, 3], [4, 5, 6, 7]]), i32([13, 40])
    q, k, v = (torch.randn(2, 5, h, 64, device=DEV).to(BF) for h in (8, 2, 2))
    a = Cache8(1, 9, 2, 16, 64, 16)
    a.all[1].fill_(100)
    b = Cache8(1, 9, 2, 16, 64, 16)
    for x, y in zip(b.all, a.all):
        x.copy_(y)
    call = lambda c: ops.rotary_append(q, k, v, c.k[0], c.v[0], tables, lens, f, None, False, 1.0, c.ks[0], c.vs[0])  # noqa: E731
    want = call(a)
    once = a.bytes()
    call(a)
    for x, y in zip(a.all, once):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = call(b)
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip((*b.all, *got), (*once, *want)):
        assert torch.equal(x, y)


def test_append_8bit_past_32_bits():
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    P = (1 << 31) // (4 * 64 * 128) + 5
    k_cache, v_cache = (torch.zeros(P, 4, 64, 128, device=DEV, dtype=torch.uint8).view(E4M3) for _ in range(2))
    ks, vs = (torch.zeros(P, 4, 4, device=DEV, dtype=torch.uint8).view(E8M0) for _ in range(2))
    k, v = (torch.randn(1, 20, 4, 128, device=DEV).to(BF) for _ in range(2))
    ops.cache_append(k, v, k_cache, v_cache, i32([[P - 1]]), i32([30]), None, None, ks, vs)
    small = Cache8(1, 1, 4, 64, 128, 16)
    for t in small.all:
        t.zero_()
    ops.cache_append(k, v, small.k[0], small.v[0], i32([[0]]), i32([30]), None, None, small.ks[0], small.vs[0])
    assert torch.equal(k_cache[-1].view(torch.uint8), small.k[0, 0].view(torch.uint8))
    assert torch.equal(vs[-1].view(torch.uint8), small.vs[0, 0].view(torch.uint8))
    assert not k_cache[:-1].view(torch.int64).any()


def test_append_nothing_to_do():
    c = Cache8(1, 4, 2, 8, 32, 8)
    was = c.bytes()
    rows = torch.randn(1, 2, 0, 2, 32, device=DEV)
    assert ops.cache_append(rows, rows, c.k, c.v, i32([[0], [1]]), i32([3, 4]), None, None, c.ks, c.vs).tolist() == [3, 4]
    none = i32([]).view(0, 3)
    assert ops.cache_append(rows[:, :0], rows[:, :0], c.k, c.v, none, i32([]), None, None, c.ks, c.vs).shape == (0,)
    q = torch.randn(2, 0, 4, 32, device=DEV)
    assert ops.rotary_append(q, rows[0], rows[0], c.k[0], c.v[0], i32([[0], [1]]), i32([3, 4]), freqs_of(32), k_scales=c.ks[0], v_scales=c.vs[0])[0].shape == (2, 0, 4, 32)
    for x, y in zip(c.all, was):
        assert torch.equal(x, y)


def test_refusals():
    x, f, at = torch.randn(2, 3, 4, 64, device=DEV).to(BF), freqs_of(64), i32([1, 2])
    for bad in (lambda: ops.rotary(x[0], at, f), lambda: ops.rotary(x, at[:1], f), lambda: ops.rotary(x, at, freqs_of(72)),
                lambda: ops.rotary(x, at, f, at)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.rotary(x.half(), at, f), lambda: ops.rotary(x, at.long(), f), lambda: ops.rotary(x, at, f.float())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(N.NklError):
        ops.rotary(x, at, freqs_of(12))
    with pytest.raises(N.NklError):
        ops.rotary(x, i32([[0] * 3] * 2), f, i32([[0] * 3] * 2))
    with pytest.raises(N.NklError):
        ops.rotary(torch.zeros(2, 129, 1, 8, device=DEV), at, freqs_of(8), torch.zeros(2, 129, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError):
        ops.rotary(x, at.cpu(), f)
    with pytest.raises(RuntimeError, match="freqs"):
        ops.rotary(x, at, f.requires_grad_())
    f = freqs_of(64)
    c, tables = Cache8(1, 4, 2, 16, 64, 16), i32([[0], [1]])
    q, k = torch.randn(2, 3, 4, 64, device=DEV).to(BF), torch.randn(2, 3, 2, 64, device=DEV).to(BF)

    def append(q=q, k=k, v=k, kc=c.k[0], vc=c.v[0], tables=tables, lens=at, f=f, count=None, ks=c.ks[0], vs=c.vs[0]):
        return ops.rotary_append(q, k, v, kc, vc, tables, lens, f, count, k_scales=ks, v_scales=vs)

    append()
    for kw in (dict(ks=None), dict(k=k[:1]), dict(v=k[:, :2]), dict(q=q[..., :32]), dict(kc=c.k), dict(ks=c.ks[0, :2]),
               dict(ks=c.ks[0, :, :, :0]), dict(tables=at), dict(lens=at[:1]), dict(count=at[:1]), dict(f=freqs_of(128))):
        with pytest.raises(ValueError):
            append(**kw)
    for kw in (dict(ks=c.all[1][0, 0]), dict(kc=c.all[0][0, 0], vc=c.all[0][1, 0]), dict(k=k.float()), dict(lens=at.long()),
               dict(ks=None, vs=None)):
        with pytest.raises(TypeError):
            append(**kw)
    for kw in (dict(kc=c.k[0].transpose(0, 1).contiguous().transpose(0, 1)), dict(ks=c.ks[0].expand(4, 2, 1).mT.contiguous().mT),
               dict(lens=at.cpu()), dict(q=q.cpu())):
        if "ks" in kw and kw["ks"].is_contiguous():
            continue
        with pytest.raises((RuntimeError, NotImplementedError)):
            append(**kw)
    odd = torch.zeros(4 * 2 * 16 * 64 + 8, dtype=torch.uint8, device=DEV)[8:].view(E4M3).view(4, 2, 16, 64)
    with pytest.raises(N.NklError):
        append(kc=odd)
    with pytest.raises(N.NklError):  # 24 entries: not whole vectors of 16
        append(q=q[..., :24], k=k[..., :24].contiguous(), v=k[..., :24].contiguous(), f=freqs_of(24),
               kc=torch.zeros(4, 2, 16, 24, device=DEV).to(E4M3), vc=torch.zeros(4, 2, 16, 24, device=DEV).to(E4M3))
    with pytest.raises(ValueError):
        ops.cache_append(k, k, c.k[0], c.v[0], tables, at, None, None, c.ks[0])
    out = append(q=q.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="rotary_append"):
        out[0].sum().backward()
