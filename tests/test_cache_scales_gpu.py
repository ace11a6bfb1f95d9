"""Forks and compactions of a cache in 8 bits: the powers of two go where their pages go."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nkilab import ops
from test_rotary_gpu import BF, DEV, E4M3, E8M0, Cache8, i32

pytestmark = pytest.mark.gpu


def pages_of(c):
    """Codes and powers of k and v as bytes, [2, layers, pages, heads, ..]."""
    return torch.stack([c.k, c.v]).view(torch.uint8), c.all[1]


# L, P, Hkv, page, d, block; the second ones' plans are a launch of their own, the odd ones' powers of two no whole vectors
SHAPES = [(2, 40, 3, 16, 32, 4), (3, 64, 8, 64, 16, 2), (1, 4099, 2, 16, 16, 16), (2, 8200, 1, 8, 16, 8), (1, 9001, 4, 8, 16, 2)]


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("L,P,Hkv,page,d,block", SHAPES)
def test_a_fork_takes_the_powers_of_its_last_page(L, P, Hkv, page, d, block, strided):
    r = np.random.RandomState(P)
    B, M = 9, 4
    c = Cache8(L, P, Hkv, page, d, block, strided)
    owned = r.permutation(P)[:B * M].reshape(B, M)
    lens = [page * M, 2 * page + 3, 0, 1, page - 1, 3 * page, page + 5, 2, page * M + 7]
    for b in range(B):
        owned[b, -(-lens[b] // page):] = -1
    owned[7, 0] = P + 3  # no page
    refs = np.zeros(P, dtype=np.int64)
    np.add.at(refs, owned[(owned >= 0) & (owned < P)], 1)
    src, dst = [1, 3, 3, 99, 4, 6, 7, 8], [2, 2, 5, 0, 4, 0, 1, 3]
    codes, powers = (t.clone() for t in pages_of(c))
    t, n, out, missing = ops.cache_fork(c.k, c.v, i32(owned.tolist()), i32(lens), i32(refs.tolist()), i32(src), i32(dst), c.ks, c.vs)
    assert missing.item() == 0
    made = {2: 1, 5: 3, 0: 6, 1: 7, 3: 8}  # the first into a slot; out of range and onto itself: none
    assert n.tolist() == [lens[made.get(b, b)] for b in range(B)]
    for to, s in made.items():
        full, rest = divmod(lens[s], page)
        if not rest or full >= M or not 0 <= owned[s, full] < P:
            continue
        fresh, from_ = int(t[to, full]), int(owned[s, full])
        assert refs[fresh] == 0
        codes[:, :, fresh, :, :rest] = codes[:, :, from_, :, :rest]
        powers[:, :, fresh] = powers[:, :, from_]
    now = pages_of(c)
    assert torch.equal(now[0], codes) and torch.equal(now[1], powers)
    # too few pages: nothing moves
    t, n, out, missing = ops.cache_fork(c.k, c.v, i32(owned.tolist()), i32(lens), i32([1] * P), i32(src), i32(dst), c.ks, c.vs)
    assert missing.item() > 0 and n.tolist() == lens
    now = pages_of(c)
    assert torch.equal(now[0], codes) and torch.equal(now[1], powers)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("L,P,Hkv,page,d,block", SHAPES)
def test_a_compaction_takes_every_moved_page_s_powers(L, P, Hkv, page, d, block, strided):
    """Pages move by `refs`: some in use are in none of the tables' rows (another table's, or held for later), and a row
    may name a page that is not in use."""
    r = np.random.RandomState(P + 1)
    c = Cache8(L, P, Hkv, page, d, block, strided)
    refs = (r.rand(P) < 0.4) * r.randint(1, 3, P)
    tables = np.full((3, 5), -1)
    used, free = np.flatnonzero(refs > 0), np.flatnonzero(refs == 0)
    tables[0, :4], tables[1, :2], tables[2, :3] = used[-4:], used[:2], [free[0], P + 9, free[-1]]
    live = len(used)
    holes, movers = [p for p in range(live) if refs[p] == 0], [p for p in range(live, P) if refs[p] > 0]
    codes, powers = (t.clone() for t in pages_of(c))
    to, from_ = torch.tensor(holes, device=DEV), torch.tensor(movers, device=DEV)
    codes[:, :, to], powers[:, :, to] = codes[:, :, from_], powers[:, :, from_]
    place = dict(zip(movers, holes))
    t, out = ops.cache_compact(c.k, c.v, i32(tables.tolist()), i32(refs.tolist()), c.ks, c.vs)
    assert t.tolist() == [[place.get(p, p) for p in row] for row in tables.tolist()]
    now = pages_of(c)
    assert torch.equal(now[0][:, :, :live], codes[:, :, :live])
    assert torch.equal(now[1][:, :, :live], powers[:, :, :live])


def test_refusals_leave_the_cache_as_it_was():
    c = Cache8(1, 6, 2, 32, 32, 16)
    tables, lens, refs = i32([[0], [-1]]), i32([5, 0]), i32([1, 0, 0, 0, 0, 1])
    was = c.bytes()

    def fork(kc=c.k, vc=c.v, ks=c.ks, vs=c.vs):
        return ops.cache_fork(kc, vc, tables, lens, refs, i32([0]), i32([1]), ks, vs)

    def compact(kc=c.k, vc=c.v, ks=c.ks, vs=c.vs):
        return ops.cache_compact(kc, vc, tables, refs, ks, vs)

    plain = torch.zeros(1, 6, 2, 32, 32, dtype=BF, device=DEV)
    turned = c.ks.mT.contiguous().mT
    assert not turned.is_contiguous()
    for op in (fork, compact):
        for kw in (dict(ks=None), dict(vs=None), dict(ks=c.ks[:, :5], vs=c.vs[:, :5]), dict(ks=c.ks[..., :1], vs=c.vs),
                   dict(ks=c.ks[0], vs=c.vs[0])):
            with pytest.raises(ValueError):
                op(**kw)
        for kw in (dict(ks=None, vs=None), dict(kc=plain, vc=plain), dict(ks=c.all[1][0], vs=c.all[1][1]), dict(vc=plain)):
            with pytest.raises(TypeError):
                op(**kw)
        for kw in (dict(ks=turned), dict(ks=c.ks.cpu(), vs=c.vs.cpu())):
            with pytest.raises(RuntimeError):
                op(**kw)
        for x, y in zip(c.all, was):
            assert torch.equal(x, y)
        assert (plain == 0).all()


def test_a_captured_fork_and_compaction_replay():
    """Another stream, and a graph that is replayed on caches filled anew: the bytes of the eager calls."""
    tables, lens, refs = i32([[7, 9, -1], [5, -1, -1], [-1, -1, -1]]), i32([21, 3, 0]), i32([0, 0, 0, 0, 0, 1, 0, 1, 0, 1])
    src, dst = i32([0, 1]), i32([2, 0])
    a, b = (Cache8(2, 10, 3, 16, 32, 4) for _ in range(2))
    start = a.bytes()

    def fill(c):
        for x, y in zip(c.all, start):
            x.copy_(y)

    def call(c):
        t, n, r, missing = ops.cache_fork(c.k, c.v, tables, lens, refs, src, dst, c.ks, c.vs)
        return (n, missing, *ops.cache_compact(c.k, c.v, t, r, c.ks, c.vs))

    want = call(a)
    fill(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(x, y) for x, y in zip(call(b), want))
        fill(b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = call(b)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        fill(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        for x, y in zip(a.all, b.all):
            assert torch.equal(x, y)
