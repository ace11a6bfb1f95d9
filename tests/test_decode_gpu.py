"""Decoding operators on the GPU against plain statements of them in 64 bits (attention) or in
Python integers (pages, verification), at the sizes and masks where they can go wrong."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from nkilab import _native as N
from nkilab import ops

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# --------------------------------------------------------------------------- attention

def visible(parents, i):
    """Token i and its ancestors; nothing for an absent token. A parent that is absent or not
    earlier counts as the root."""
    if parents[i] < -1:
        return []
    seen, at = [i], i
    while 0 <= parents[at] < at and parents[parents[at]] >= -1:
        at = parents[at]
        seen.append(at)
    return seen


def attention_64(q, k, v, kc, vc, tables, lens, parents, scale):
    """(out, sum of p |v|) in 64 bits."""
    B, T, H, d = q.shape
    P, Hkv, page, _ = kc.shape
    out = torch.zeros(B, T, H, d, dtype=torch.float64)
    mag = torch.zeros_like(out)
    q, k, v = (t.double().cpu() for t in (q, k, v))
    tables, lens = tables.cpu().tolist(), lens.cpu().tolist()
    trees = parents.cpu().tolist() if parents is not None else [list(range(-1, T - 1))] * B
    for b in range(B):
        n = lens[b]
        pages = torch.tensor(tables[b][:-(-n // page)], dtype=torch.long, device=kc.device)
        old_k, old_v = (c[pages].double().cpu().transpose(1, 2).reshape(-1, Hkv, d)[:n] for c in (kc, vc))
        for i in range(T):
            see = visible(trees[b], i)
            if not see:
                continue
            for h in range(H):
                g = h // (H // Hkv)
                ks, vs = torch.cat([old_k[:, g], k[b, see, g]]), torch.cat([old_v[:, g], v[b, see, g]])
                p = (ks @ q[b, i, h] * scale).softmax(0)
                out[b, i, h], mag[b, i, h] = p @ vs, p @ vs.abs()
    return out, mag


def check_attention(got, want, mag):
    """fp32: sums of d products and n exponentials, each within some 2^-24 of its size. bf16:
    the output's rounding (2^-9 of it) and that of the exponentials (2^-9 of each, so at most
    2^-9 sum p |v|), with 5 % for the products of the two and fp32's part."""
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    err = (got - want).abs()
    bound = 2e-5 * (1 + mag)
    if BF_LIKE[0]:
        bound = bound + 1.05 * 2.0 ** -9 * (want.abs() + mag)
    assert (err <= bound).all(), float((err / bound).max())


BF_LIKE = [False]


def setup_attention(B, T, H, Hkv, d, page, lens, dtype, seed=0, layout="heads", spare=3, junk=float("nan")):
    """Inputs whose cache holds `junk` wherever no sequence looks."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = np.random.RandomState(seed)
    M = max(1, max(-(-n // page) for n in lens)) + 1
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    order, at = r.permutation(P), 0
    shape = (P, Hkv, page, d) if layout == "heads" else (P, page, Hkv, d)
    kc, vc = (torch.full(shape, junk, device=DEV, dtype=dtype) for _ in range(2))
    if layout != "heads":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    tables = np.full((B, M), -1)
    for b, n in enumerate(lens):
        tables[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        for p in range(need[b]):
            used = min(page, n - p * page)
            for c in (kc, vc):
                c[int(tables[b, p]), :, :used] = torch.randn(Hkv, used, d, generator=g, device=DEV).to(dtype)
    qkv = torch.randn(B, T, H + 2 * Hkv, d, generator=g, device=DEV).to(dtype)
    q, k, v = qkv.split([H, Hkv, Hkv], 2)
    BF_LIKE[0] = dtype == BF
    return q, k, v, kc, vc, i32(tables), i32(lens)


def random_trees(r, B, T, absent=0.2):
    parents = np.full((B, T), -1)
    for b in range(B):
        for i in range(1, T):
            parents[b, i] = -2 if r.rand() < absent else r.randint(-1, i)
    return parents


ATTENTION = [
    # B, T, H, Hkv, d, page, lens, dtype
    (1, 1, 8, 8, 128, 16, [0], BF),                      # nothing cached: a token sees itself
    (1, 1, 8, 2, 128, 16, [1], BF),
    (1, 1, 32, 8, 128, 64, [2000], BF),
    (3, 1, 4, 4, 64, 8, [127, 128, 129], BF),            # at a tile's edge
    (4, 5, 8, 1, 64, 16, [0, 1, 300, 1025], BF),
    (2, 16, 8, 8, 128, 64, [700, 63], BF),
    (3, 33, 12, 4, 128, 32, [65, 511, 0], BF),           # 99 rows of a key/value head: 42 tokens to a tile
    (2, 64, 8, 2, 128, 128, [513, 1000], BF),            # 256 rows
    (2, 128, 4, 1, 128, 256, [900, 40], BF),             # 512 rows
    (1, 128, 2, 2, 64, 24, [777], BF),                   # pages that end inside a tile
    (2, 3, 10, 2, 128, 48, [1000, 95], BF),              # 5 heads share
    (1, 2, 96, 1, 64, 16, [400], BF),                    # 96 heads share
    (1, 2, 160, 1, 64, 16, [200], BF),                   # 160 heads share
    (2, 3, 4, 2, 96, 16, [50, 200], BF),                 # head_dim of the CUDA-core kernel
    (2, 3, 4, 2, 64, 17, [50, 200], BF),                 # odd pages
    (2, 7, 8, 4, 64, 24, [0, 999], F32),
    (1, 1, 8, 8, 128, 16, [3000], F32),
    (2, 40, 6, 2, 128, 64, [129, 5], F32),
    (3, 2, 3, 3, 8, 1, [0, 1, 33], F32),
]


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("B,T,H,Hkv,d,page,lens,dtype", ATTENTION)
def test_attention_tree(B, T, H, Hkv, d, page, lens, dtype, tree):
    x = setup_attention(B, T, H, Hkv, d, page, lens, dtype, seed=B + T + d)
    parents = i32(random_trees(np.random.RandomState(T), B, T)) if tree else None
    got = ops.attention_tree(*x, parents)
    assert got.shape == x[0].shape and got.dtype == dtype and got.is_contiguous()
    check_attention(got, *attention_64(*x, parents, 1 / math.sqrt(d)))
    N.check_device(torch.cuda.current_stream().cuda_stream)


def cancelling(B, T, H, Hkv, d, page, lens):
    """Peaked weights over values of one size and alternating sign: |out| is far below sum p |v|."""
    x = list(setup_attention(B, T, H, Hkv, d, page, lens, BF, seed=sum(lens)))
    x[0] = x[0] * 3
    x[2] = (1 - 2 * (torch.arange(T, device=DEV) % 2))[None, :, None, None].expand_as(x[2]).to(BF)
    for b, n in enumerate(lens):
        for p in range(-(-n // page)):
            used = min(page, n - p * page)
            x[4][int(x[5][b, p]), :, :used] = (1 - 2 * ((torch.arange(used, device=DEV) + p * page) % 2))[:, None].to(BF)
    return x


@pytest.mark.parametrize("T,H,d,page,lens", [(1, 8, 128, 16, [5, 60, 300, 1024]), (9, 8, 64, 16, [0, 33, 129, 1024]),
                                             (64, 16, 128, 64, [20, 900, 1024]), (100, 4, 64, 24, [77, 1000])])
def test_attention_keeps_the_exponentials_second_part(T, H, d, page, lens):
    """bf16, up to 1024 cached positions: the first part of an exponential is cut off (less than
    2^-7 of it is left), the second is that, rounded (2^-8 of it). So the error is the output's
    rounding (2^-8 of it), at most 2^-15 sum p |v|, and fp32's part."""
    x = cancelling(len(lens), T, H, 2, d, page, lens)
    want, mag = attention_64(*x, None, 1 / math.sqrt(d))
    err = (ops.attention_tree(*x).double().cpu() - want).abs()
    bound = 2e-5 * (1 + mag) + (1 + 2.0 ** -6) * 2.0 ** -8 * want.abs() + 2.0 ** -15 * mag
    assert (err <= bound).all(), float((err / bound).max())


def test_attention_past_the_exponentials_second_part():
    x = cancelling(2, 3, 8, 2, 128, 16, [1025, 1024])
    check_attention(ops.attention_tree(*x), *attention_64(*x, None, 128 ** -0.5))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_odd_parents(dtype):
    """Parents that are no earlier token, children of absent tokens, a whole slot absent, a
    chain as long as the limit."""
    x = setup_attention(4, 128, 2, 1, 64, 16, [20, 300, 0, 7], dtype)
    parents = np.full((4, 128), -1)
    parents[0] = np.arange(-1, 127)
    parents[1, :6] = [-1, 5, 1, -2, 3, 4]
    parents[1, 6:] = 200
    parents[2] = -2
    parents[3] = np.maximum(np.arange(128) // 2 - 1, -1)
    parents[3, 40:] = -7
    parents = i32(parents)
    got = ops.attention_tree(*x, parents)
    check_attention(got, *attention_64(*x, parents, 1 / 8))
    assert (got[2] == 0).all() and (got[3, 40:] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_layouts(dtype):
    """A cache with positions before heads, a layer of a larger cache, tensors of odd strides."""
    x = setup_attention(2, 4, 8, 2, 64, 16, [90, 33], dtype, layout="positions")
    want = attention_64(*x, None, 0.3)
    check_attention(ops.attention_tree(*x, None, 0.3), *want)
    q, k, v, kc, vc, tables, lens = x
    big_k, big_v = (torch.full((3, *c.shape), float("nan"), device=DEV, dtype=dtype) for c in (kc, vc))
    big_k[1], big_v[1] = kc, vc
    check_attention(ops.attention_tree(q, k, v, big_k[1], big_v[1], tables, lens, None, 0.3), *want)
    odd = torch.empty(2, 4, 8, 67, device=DEV, dtype=dtype)[..., 1:65]  # rows that start anywhere
    odd.copy_(q)
    kt = k.transpose(1, 2).contiguous().transpose(1, 2)  # strides other than v's
    check_attention(ops.attention_tree(odd, kt, v, kc, vc, tables, lens, None, 0.3), *want)


def shifted(t):
    """The same values, contiguous, one element past an aligned address."""
    buf = torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)
    buf[1:] = t.flatten()
    return buf[1:].view(t.shape)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_unaligned_inputs(dtype):
    """Contiguous tensors that begin anywhere are taken as their aligned copies are."""
    q, k, v, kc, vc, tables, lens = setup_attention(2, 3, 8, 2, 64, 16, [90, 33], dtype, junk=0.0)
    want = ops.attention_tree(q, k, v, kc, vc, tables, lens)
    for a, b, c in ((shifted(q), k, v), (q, shifted(k), v), (q, k.contiguous(), shifted(v)), (shifted(q), shifted(k), shifted(v))):
        assert torch.equal(ops.attention_tree(a, b, c, kc, vc, tables, lens), want)
    lens = lens - 3
    for a, b in ((shifted(k), shifted(v)), (k.contiguous(), shifted(v))):
        got, want = (kc.clone(), vc.clone()), (kc.clone(), vc.clone())
        ops.cache_append(a, b, *got, tables, lens)
        ops.cache_append(k, v, *want, tables, lens)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attention_extreme_scores():
    """Scores that leave one key, and lowest values in masked places."""
    q, k, v, kc, vc, tables, lens = setup_attention(2, 8, 4, 2, 128, 16, [300, 17], BF, junk=-3.3e38)
    q = q * 40
    parents = i32(random_trees(np.random.RandomState(1), 2, 8))
    check_attention(ops.attention_tree(q, k, v, kc, vc, tables, lens, parents),
                    *attention_64(q, k, v, kc, vc, tables, lens, parents, 128 ** -0.5))


@pytest.mark.parametrize("dtype,H", [(BF, 4), (BF, 40), (F32, 4)])
def test_attention_infinities_of_unseen_tokens(dtype, H):
    """Infinities and NaN in the k and v of absent tokens, and of tokens on other branches, leave
    no trace; a token's own show in its row and its descendants'."""
    q, k, v, kc, vc, tables, lens = setup_attention(2, 9, H, 2, 64, 16, [300, 0], dtype)
    parents = [[-1, 0, 0, 2, -1, -2, 4, 3, -2], [-1, -1, 1, 2, 3, -2, -2, 1, 7]]
    k, v = k.clone(), v.clone()
    k[0, 5], v[0, 5] = float("nan"), float("nan")  # absent
    v[0, 8] = float("inf")
    v[1, 5], k[1, 6] = float("-inf"), float("inf")
    clean = [t.clone() for t in (k, v)]
    v[0, 2, 0, 3], v[0, 2, 1, 60] = float("inf"), float("nan")  # seen by 2, 3 and 7
    v[1, 0, 0, :] = float("-inf")  # a leaf
    x = (q, k, v, kc, vc, tables, lens)
    for ks in (k, clean[0]):
        ks[0, 5], ks[1, 6] = 0, 0  # the statement in 64 bits never looks at them, but copies
    want, mag = attention_64(q, *clean, kc, vc, tables, lens, i32(parents), 1 / 8)
    k[0, 5], k[1, 6] = float("nan"), float("inf")
    got = ops.attention_tree(*x, i32(parents))
    shows = torch.zeros(2, 9, H, 64, dtype=torch.bool)
    shows[0, [2, 3, 7], :H // 2, 3] = True
    shows[0, [2, 3, 7], H // 2:, 60] = True
    shows[1, 0, :H // 2] = True
    shows = shows.to(DEV)
    assert not torch.isfinite(got[shows]).any()
    assert (got[0, [2, 3, 7], :H // 2, 3] == float("inf")).all() and got[0, [2, 3, 7], H // 2:, 60].isnan().all()
    check_attention(torch.where(shows, 0, got), torch.where(shows.cpu(), 0, want), mag)


def put(x, b, pos, head, col, k=None, v=None):
    """Sets one element of a cached position's key or value."""
    kc, vc, tables, page = x[3], x[4], x[5], x[3].shape[2]
    at = int(tables[b, pos // page]), head, pos % page, col
    for c, value in ((kc, k), (vc, v)):
        if value is not None:
            c[at] = value


def check_with_infinities(got, want, mag):
    """Infinities and NaN where the statement in 64 bits has them, the rest as ever."""
    got, finite = got.cpu(), torch.isfinite(want)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()].double(), want[want.isinf()])
    check_attention(torch.where(finite, got, 0), torch.where(finite, want, 0), torch.where(finite, mag, 0))


INFINITIES = [(F32, 64, 16), (F32, 128, 24), (BF, 96, 16), (BF, 64, 17), (BF, 64, 16), (BF, 128, 24)]


@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("dtype,d,page", INFINITIES)
def test_attention_infinities_in_the_cache(dtype, d, page, T):
    """Infinities, NaN and the largest values in cached positions show as the formula has them: an
    infinite value in its column, a key whose score is minus infinity not at all."""
    inf, big = float("inf"), torch.finfo(dtype).max
    if dtype == BF and d != 96 and page % 8 == 0:
        big /= 1024  # weights of up to 2^8 and their sum are divided out last
    x = list(setup_attention(4, T, 4, 2, d, page, [130, 700, 90, 300], dtype, seed=d))
    q = x[0] = x[0].clone()
    q[..., 0] = q[..., 0].abs() + 0.25
    for pos, col, v in ((5, 3, inf), (120, 3, inf), (10, 7, inf), (90, 7, -inf), (2, 9, float("nan")), (129, 11, -inf)):
        put(x, 0, pos, 0, col, v=v)
    put(x, 0, 20, 0, 0, k=-inf)
    put(x, 1, 699, 0, 0, k=-inf)
    put(x, 1, 7, 1, 0, k=inf)  # the rows of this head are NaN
    put(x, 1, 300, 0, d - 1, v=-inf)
    for pos, col, v in ((3, 5, big), (4, 6, -big)):
        put(x, 2, pos, 1, col, v=v)
    put(x, 3, 4, 0, 1, k=big)
    q[3, :, :2] *= 1e-37  # its score is at most of the size of 1
    check_with_infinities(ops.attention_tree(*x, None), *attention_64(*x, None, 1 / math.sqrt(d)))


@pytest.mark.parametrize("T", [1, 70])
@pytest.mark.parametrize("dtype,d,page", INFINITIES)
def test_attention_nan_scores_alone(dtype, d, page, T):
    """Keys that are all NaN, where the rest of the row is finite: in eight keys in a row, in the
    first tiles of a long row (some of them a piece by themselves), in all that a token sees."""
    x = list(setup_attention(3, T, 8, 8, d, page, [4096, 64, 0], dtype, seed=d + T))
    for head in range(8):
        for pos in range(128 * (head + 1)):
            put(x, 0, pos, head, 0, k=float("nan"))
    for pos in range(8, 16):
        put(x, 1, pos, 1, 5, k=float("nan"))
        put(x, 1, pos + 32, 1, 5, k=float("nan"))
    x[1] = x[1].clone()
    x[1][2, 0, 0] = float("nan")  # seen by every token after it
    check_with_infinities(ops.attention_tree(*x, None), *attention_64(*x, None, 1 / math.sqrt(d)))


@pytest.mark.parametrize("dtype,d,page", INFINITIES)
def test_attention_scores_of_minus_infinity_alone(dtype, d, page):
    """A token that sees nothing but keys scored minus infinity is 0 / 0, whichever kernel takes it
    and however its row is cut; an absent one is 0."""
    q, k, v, kc, vc, tables, lens = setup_attention(3, 3, 4, 2, d, page, [0, 40, 3000], dtype, junk=0.0)
    q[..., 0] = 1
    for c in (k, kc):
        c[..., 0] = float("-inf")
    x = (q, k, v, kc, vc, tables, lens)
    parents = i32([[-1, 0, -2]] * 3)
    got = ops.attention_tree(*x, parents)
    assert got[:, :2].isnan().all() and (got[:, 2] == 0).all()


@pytest.mark.parametrize("dtype,T", [(BF, 1), (BF, 70), (F32, 3)])
def test_attention_growing_maxima(dtype, T):
    """Every later key scores higher: the running maximum grows in every tile."""
    q, k, v, kc, vc, tables, lens = setup_attention(1, T, 2, 1, 64, 16, [1500], dtype)
    q = torch.ones_like(q)
    ramp = torch.arange(tables.numel() * 16, device=DEV).float()[:1500] / 40
    for p in range(-(-1500 // 16)):
        part = ramp[p * 16:(p + 1) * 16]
        kc[int(tables[0, p]), 0, :part.numel()] = (part[:, None] / 8).expand(-1, 64).to(dtype)
    x = (q, k, v, kc, vc, tables, lens)
    check_attention(ops.attention_tree(*x, None), *attention_64(*x, None, 1 / 8))


def test_attention_many_short_and_one_long():
    """Ragged lengths, so that the blocks' shares begin and end anywhere."""
    lens = [3000] + [0, 1, 5, 130, 64] * 12 + [1111]
    x = setup_attention(len(lens), 3, 4, 2, 64, 16, lens, BF)
    check_attention(ops.attention_tree(*x, None), *attention_64(*x, None, 1 / 8))


def test_attention_wide_batch():
    """More sequences than a block has threads."""
    lens = [(7 * b) % 41 for b in range(700)]
    x = setup_attention(len(lens), 1, 2, 1, 64, 8, lens, BF)
    check_attention(ops.attention_tree(*x, None), *attention_64(*x, None, 1 / 8))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_offsets_past_32_bits(dtype):
    """Pages at the far end of a cache of more than 2^31 elements."""
    page, Hkv, d = 64, 8, 128
    P = (1 << 31) // (page * Hkv * d) + 40
    kc, vc = (torch.empty(P, Hkv, page, d, device=DEV, dtype=dtype) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(0)
    tables = i32([[P - 1, 3, P - 7, -1]])
    for p in (P - 1, 3, P - 7):
        for c in (kc, vc):
            c[p] = torch.randn(Hkv, page, d, generator=g, device=DEV).to(dtype)
    q, k, v = (torch.randn(1, 2, h, d, generator=g, device=DEV).to(dtype) for h in (16, Hkv, Hkv))
    BF_LIKE[0] = dtype == BF
    x = (q, k, v, kc, vc, tables, i32([150]))
    check_attention(ops.attention_tree(*x, None), *attention_64(*x, None, d ** -0.5))


def test_attention_tables_out_of_range_are_harmless():
    """A table that names no page reads zeros; other sequences are untouched."""
    x = list(setup_attention(2, 2, 4, 2, 64, 16, [100, 100], BF, junk=0.0))
    want, mag = attention_64(*x, None, 1 / 8)
    x[5] = x[5].clone()
    x[5][1, :7] = i32([-1, 1 << 30, -5, 999999, -1, -2147483648, 77777])
    x[6] = i32([100, 1 << 29])
    got = ops.attention_tree(*x, None)
    check_attention(got[:1], want[:1], mag[:1])


@pytest.mark.parametrize("dtype,T", [(BF, 1), (BF, 64), (F32, 5)])
def test_attention_repeats_streams_and_graphs(dtype, T):
    """The same bits on every launch, on another stream, and when a graph replays with lengths
    that have changed since the capture."""
    x = setup_attention(4, T, 8, 2, 128, 16, [900, 3, 0, 2049], dtype, junk=0.0)
    a = ops.attention_tree(*x, None)
    for _ in range(3):
        assert torch.equal(ops.attention_tree(*x, None), a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = ops.attention_tree(*x, None)
    side.synchronize()
    assert torch.equal(a, b)
    lens = x[6].clone()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c = ops.attention_tree(*x[:6], lens, None)
    lens.copy_(i32([17, 3, 0, 1024]))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, ops.attention_tree(*x[:6], lens, None))
    lens.copy_(x[6])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, a)


def test_attention_refusals():
    x = list(setup_attention(2, 3, 4, 2, 64, 16, [10, 20], BF))

    def bad(error, **change):
        names = ["q", "k", "v", "kc", "vc", "tables", "lens"]
        y = [change.get(n, t) for n, t in zip(names, x)]
        with pytest.raises(error):
            ops.attention_tree(*y, change.get("parents"))

    q, k, v, kc, vc, tables, lens = x
    bad(ValueError, q=q[..., :32])
    bad(ValueError, q=q[:, :, :3])
    bad(ValueError, k=k[:1], v=v[:1])
    bad(TypeError, q=q.float())
    bad(TypeError, vc=vc.float())
    bad(TypeError, lens=lens.long())
    bad(TypeError, tables=tables.long())
    bad(ValueError, lens=lens[:1])
    bad(ValueError, parents=i32([[0, 0], [0, 0]]))
    bad(RuntimeError, lens=lens.cpu())
    bad(RuntimeError, vc=vc.transpose(2, 3).contiguous().transpose(2, 3))
    bad(ValueError, kc=kc[None])
    bad(TypeError, q=q.half(), k=k.half(), v=v.half(), kc=kc.half(), vc=vc.half())
    with pytest.raises(NotImplementedError):
        ops.attention_tree(*(t.cpu() for t in x))
    y = setup_attention(1, 129, 2, 2, 64, 16, [10], BF)
    with pytest.raises(ValueError, match="129"):
        ops.attention_tree(*y)
    z = [torch.zeros(1, 1, 2, 68, device=DEV, dtype=BF)] * 3 + [torch.zeros(2, 2, 16, 68, device=DEV, dtype=BF)] * 2
    with pytest.raises(N.NklError, match="head_dim"):
        ops.attention_tree(*z, i32([[0]]), i32([3]))


def test_attention_nothing_to_do():
    x = setup_attention(2, 3, 4, 2, 64, 16, [10, 20], BF)
    q, k, v, kc, vc, tables, lens = x
    assert ops.attention_tree(q[:, :0], k[:, :0], v[:, :0], kc, vc, tables, lens).shape == (2, 0, 4, 64)
    assert ops.attention_tree(q[:0], k[:0], v[:0], kc, vc, tables[:0], lens[:0]).shape == (0, 3, 4, 64)


# --------------------------------------------------------------------------- pages

class Model:
    """The cache in Python: what each operation is to do."""

    def __init__(self, tables, lens, refs, page):
        self.t, self.n, self.r, self.page = [list(r) for r in tables], list(lens), list(refs), page

    def free_pages(self):
        return [p for p, c in enumerate(self.r) if c == 0]

    def drop(self, b):
        for p in self.t[b]:
            if 0 <= p < len(self.r):
                self.r[p] -= 1
        self.t[b], self.n[b] = [-1] * len(self.t[b]), 0

    def check(self, tables, lens, refs):
        assert tables.tolist() == self.t and refs.tolist() == self.r
        if lens is not None:
            assert lens.tolist() == self.n


def pool(L, B, P, Hkv, page, d, lens, dtype=BF, M=None, seed=0, layout="heads"):
    r = np.random.RandomState(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    M = M or max(-(-n // page) for n in lens) + 2
    order, at = r.permutation(P), 0
    tables, refs = np.full((B, M), -1), np.zeros(P, int)
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            tables[b, i] = order[at]
            refs[order[at]] += 1
            at += 1
    shape = (L, P, Hkv, page, d) if layout == "heads" else (L, P, page, Hkv, d)
    kc, vc = (torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2))
    if layout != "heads":
        kc, vc = kc.transpose(2, 3), vc.transpose(2, 3)
    return kc, vc, i32(tables), i32(lens), i32(refs)


POOLS = [dict(L=1, B=4, P=20, Hkv=2, page=8, d=64, lens=[0, 1, 16, 33]),
         dict(L=3, B=5, P=40, Hkv=1, page=24, d=128, lens=[24, 100, 0, 71, 48]),
         dict(L=2, B=3, P=9, Hkv=4, page=17, d=8, lens=[18, 0, 34], dtype=F32),
         dict(L=2, B=4, P=30, Hkv=2, page=16, d=64, lens=[15, 0, 160, 17], layout="positions"),
         dict(L=1, B=2, P=3000, Hkv=1, page=1, d=8, lens=[900, 0])]


@pytest.mark.parametrize("at", range(len(POOLS)))
@pytest.mark.parametrize("T", [1, 7, 300])
def test_append(at, T):
    c = dict(POOLS[at])
    lens = c["lens"]
    c["P"] = sum(-(-(n + T) // c["page"]) for n in lens) + 2
    full = [n + T for n in lens]
    kc, vc, tables, _, _ = pool(**{**c, "lens": full})
    r = np.random.RandomState(T)
    L, B, Hkv, d = c["L"], c["B"], c["Hkv"], c["d"]
    both = torch.randn(L, B, T, 2, Hkv, d, device=DEV).to(kc.dtype)
    k, v = both[:, :, :, 0], both[:, :, :, 1]
    for picked in (False, True):
        count = [T] * B
        path = [list(range(T))] * B
        if picked:
            count = [int(r.randint(0, T + 1)) for _ in range(B)]
            count[0] = 0
            path = [sorted(r.choice(T, m, replace=False).tolist()) + [-1] * (T - m) for m in count]
        want_k, want_v = kc.clone(), vc.clone()
        t = tables.tolist()
        for b in range(B):
            for j in range(count[b]):
                p, s = divmod(lens[b] + j, c["page"])
                want_k[:, t[b][p], :, s], want_v[:, t[b][p], :, s] = k[:, b, path[b][j]], v[:, b, path[b][j]]
        out = ops.cache_append(k, v, kc, vc, tables, i32(lens), i32(path) if picked else None, i32(count) if picked else None)
        assert out.tolist() == [n + m for n, m in zip(lens, count)]
        assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_append_drops_rows_without_a_page():
    kc, vc, tables, lens, _ = pool(1, 3, 8, 1, 8, 64, [8, 3, 0], M=2)
    tables[2] = i32([5000, -9])
    want_k, want_v = kc.clone(), vc.clone()
    k, v = (torch.randn(1, 3, 20, 1, 64, device=DEV).to(BF) for _ in range(2))
    p = int(tables[1, 0])
    want_k[0, p, 0, 3:8], want_v[0, p, 0, 3:8] = k[0, 1, :5, 0], v[0, 1, :5, 0]
    path = torch.arange(20, dtype=torch.int32, device=DEV).repeat(3, 1)
    path[1, 1] = 99  # no such row
    want_k[0, p, 0, 4], want_v[0, p, 0, 4] = kc[0, p, 0, 4], vc[0, p, 0, 4]
    out = ops.cache_append(k, v, kc, vc, tables, lens, path, i32([20, 20, 25]))
    assert out.tolist() == [28, 23, 20]
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


@pytest.mark.parametrize("at", range(len(POOLS)))
def test_reserve(at):
    c = POOLS[at]
    kc, vc, tables, lens, refs = pool(**c, M=max(-(-n // c["page"]) for n in c["lens"]) + 3)
    extra = [(5 * b + 2) % (2 * c["page"] + 1) for b in range(c["B"])]
    m = Model(tables.tolist(), c["lens"], refs.tolist(), c["page"])
    free = m.free_pages()
    want = 0
    for b in range(c["B"]):
        have = sum(p >= 0 for p in m.t[b])
        for i in range(have, -(-(m.n[b] + extra[b]) // c["page"])):
            want += 1
            if free:
                m.t[b][i] = free.pop(0)
                m.r[m.t[b][i]] = 1
    t, r, missing = ops.cache_reserve(tables, lens, refs, i32(extra), c["page"])
    assert want <= len(Model(tables.tolist(), c["lens"], refs.tolist(), 1).free_pages())
    assert missing.item() == 0
    m.check(t, None, r)


def test_reserve_all_or_nothing():
    kc, vc, tables, lens, refs = pool(1, 3, 8, 1, 8, 64, [8, 3, 0], M=4)
    t, r, missing = ops.cache_reserve(tables, lens, refs, i32([24, 24, 24]), 8)  # 3 + 3 + 3 pages, 6 free
    assert missing.item() == 3 and torch.equal(t, tables) and torch.equal(r, refs)
    t, r, missing = ops.cache_reserve(tables, lens, refs, i32([0, 40, 0]), 8)  # more than a row holds
    assert missing.item() == 2 and torch.equal(t, tables) and torch.equal(r, refs)
    t, r, missing = ops.cache_reserve(tables, lens, refs, i32([0, -5, 0]), 8)
    assert missing.item() == 0 and torch.equal(t, tables) and torch.equal(r, refs)


def expect_fork(m, kc, vc, src, dst):
    page, B = m.page, len(m.n)
    forks, taken = [], set()
    for s, t in zip(src, dst):
        if 0 <= s < B and 0 <= t < B and s != t and t not in taken:
            taken.add(t)
            forks.append((s, t))
    free, old_t, old_n = m.free_pages(), [list(r) for r in m.t], list(m.n)
    lack = max(0, sum(old_n[s] % page > 0 for s, _ in forks) - len(free))
    if lack:
        return lack
    for s, t in forks:
        m.drop(t)
    for s, t in forks:
        full, rest = divmod(old_n[s], page)
        row = old_t[s][:full]
        if rest:
            p = free.pop(0)
            for c in (kc, vc):
                c[:, p, :, :rest] = c[:, old_t[s][full], :, :rest].clone()
            row = row + [p]
        for p in row:
            m.r[p] += 1
        m.t[t], m.n[t] = row + [-1] * (len(old_t[s]) - len(row)), old_n[s]
    return 0


@pytest.mark.parametrize("at", range(len(POOLS)))
@pytest.mark.parametrize("src,dst", [([0], [1]), ([1, 1, 0], [0, 0, 1]), ([0, 1], [1, 0]), ([], []),
                                     ([0, -1, 99, 1, 0], [0, 1, 1, -2, 77])])
def test_fork(at, src, dst):
    c = POOLS[at]
    kc, vc, tables, lens, refs = pool(**c)
    m, want_k, want_v = Model(tables.tolist(), c["lens"], refs.tolist(), c["page"]), kc.clone(), vc.clone()
    lack = expect_fork(m, want_k, want_v, src, dst)
    t, n, r, missing = ops.cache_fork(kc, vc, tables, lens, refs, i32(src), i32(dst))
    assert missing.item() == lack
    m.check(t, n, r)
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_fork_all_or_nothing():
    kc, vc, tables, lens, refs = pool(2, 4, 5, 1, 8, 64, [20, 9, 0, 0])  # 5 pages, all taken
    a, b = kc.clone(), vc.clone()
    t, n, r, missing = ops.cache_fork(kc, vc, tables, lens, refs, i32([0, 1]), i32([2, 3]))
    assert missing.item() == 2
    for x, y in ((t, tables), (n, lens), (r, refs), (kc, a), (vc, b)):
        assert torch.equal(x, y)


def test_fork_many():
    """More forks and pages than a block has threads, shared and freed again."""
    B, P = 2500, 4000
    lens = [11, 16, 5] + [0] * (B - 3)
    kc, vc, tables, n, refs = pool(1, B, P, 1, 8, 8, lens, M=3)
    src, dst = [i % 3 for i in range(B - 3)], list(range(3, B))
    m, want_k, want_v = Model(tables.tolist(), lens, refs.tolist(), 8), kc.clone(), vc.clone()
    assert expect_fork(m, want_k, want_v, src, dst) == 0
    t, n, r, missing = ops.cache_fork(kc, vc, tables, n, refs, i32(src), i32(dst))
    assert missing.item() == 0
    m.check(t, n, r)
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    gone = list(range(0, B, 2))
    for b in gone:
        m.drop(b)
    t, n, r = ops.cache_free(t, n, r, i32(gone))
    m.check(t, n, r)


@pytest.mark.parametrize("at", range(len(POOLS)))
@pytest.mark.parametrize("slots", [[], [0], [1, 0, 1], [-1, 99, 1]])
def test_free_and_compact(at, slots):
    c = POOLS[at]
    kc, vc, tables, lens, refs = pool(**c)
    m = Model(tables.tolist(), c["lens"], refs.tolist(), c["page"])
    for b in {s for s in slots if 0 <= s < c["B"]}:
        m.drop(b)
    t, n, r = ops.cache_free(tables, lens, refs, i32(slots))
    m.check(t, n, r)
    live = [p for p, x in enumerate(m.r) if x > 0]
    holes = [p for p in range(len(live)) if m.r[p] <= 0]
    move = dict(zip([p for p in live if p >= len(live)], holes))
    want_k, want_v = kc.clone(), vc.clone()
    for a, b in move.items():
        want_k[:, b], want_v[:, b] = kc[:, a], vc[:, a]
        m.r[b], m.r[a] = m.r[a], 0
    m.t = [[move.get(p, p) for p in row] for row in m.t]
    t, r = ops.cache_compact(kc, vc, t, r)
    m.check(t, None, r)
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_compact_wide():
    """Thousands of pages, most of them free."""
    r = np.random.RandomState(3)
    P = 9001
    refs = (r.rand(P) < 0.3) * r.randint(1, 4, P)
    kc = torch.arange(P, device=DEV, dtype=F32).view(1, P, 1, 1, 1).expand(2, P, 1, 1, 4).contiguous()
    vc = kc + 0.5
    tables = i32(np.where(refs > 0, np.arange(P), -1).reshape(1, P))
    t, out = ops.cache_compact(kc, vc, tables, i32(refs))
    live = int((refs > 0).sum())
    assert (out[:live] > 0).all() and (out[live:] == 0).all()
    at = t[0][torch.from_numpy(refs > 0).to(DEV)].long()
    assert sorted(at.tolist()) == list(range(live))
    assert torch.equal(kc[1, at, 0, 0, 0].long().cpu(), torch.from_numpy(np.flatnonzero(refs)))
    assert torch.equal(vc[0, at, 0, 0, 3], kc[1, at, 0, 0, 0] + 0.5)
    assert torch.equal(out[at].cpu(), torch.from_numpy(refs[refs > 0]).int())


def test_page_operations_past_32_bits():
    """Copies between the ends of caches of more than 2^32 bytes."""
    page, Hkv, d = 64, 8, 128
    P = (1 << 31) // (page * Hkv * d) + 5
    kc, vc = (torch.zeros(1, P, Hkv, page, d, device=DEV, dtype=BF) for _ in range(2))
    kc[0, P - 1], vc[0, P - 1] = 3.0, 4.0
    refs = torch.zeros(P, dtype=torch.int32, device=DEV)
    refs[P - 1] = 1
    t, n, r, missing = ops.cache_fork(kc, vc, i32([[P - 1], [-1]]), i32([40, 0]), refs, i32([0]), i32([1]))
    assert t.tolist() == [[P - 1], [0]] and r[0] == 1
    assert (kc[0, 0, :, :40] == 3).all() and (kc[0, 0, :, 40:] == 0).all() and (vc[0, 0, :, :40] == 4).all()
    t, r = ops.cache_compact(kc, vc, t, r)
    assert t.tolist() == [[1], [0]] and r[:3].tolist() == [1, 1, 0]
    assert (kc[0, 1] == 3).all() and (vc[0, 1] == 4).all()


def test_page_refusals():
    kc, vc, tables, lens, refs = pool(1, 3, 8, 1, 8, 64, [8, 3, 0])
    k = torch.zeros(1, 3, 2, 1, 64, device=DEV, dtype=BF)
    with pytest.raises(ValueError):
        ops.cache_append(k[:, :, :, :, :32], k[:, :, :, :, :32], kc, vc, tables, lens)
    with pytest.raises(TypeError):
        ops.cache_append(k.float(), k.float(), kc, vc, tables, lens)
    with pytest.raises(ValueError):
        ops.cache_append(k, k, kc, vc, tables, lens, count=i32([1]))
    with pytest.raises(TypeError):
        ops.cache_append(k, k, kc, vc, tables, lens.long())
    with pytest.raises(ValueError):
        ops.cache_fork(kc, vc, tables, lens, refs[:4], i32([0]), i32([1]))
    with pytest.raises(ValueError):
        ops.cache_fork(kc, vc, tables, lens, refs, i32([0]), i32([1, 2]))
    with pytest.raises(RuntimeError):
        ops.cache_fork(kc, vc.transpose(3, 4).contiguous().transpose(3, 4), tables, lens, refs, i32([0]), i32([1]))
    with pytest.raises(TypeError):
        ops.cache_free(tables, lens, refs, torch.tensor([0], device=DEV))
    with pytest.raises(RuntimeError):
        ops.cache_compact(kc, vc, tables.t().contiguous().t(), refs)
    with pytest.raises(N.NklError, match="pages"):
        ops.cache_reserve(tables, lens, refs, lens, 0)
    with pytest.raises(NotImplementedError):
        ops.cache_free(tables.cpu(), lens.cpu(), refs.cpu(), torch.tensor([0], dtype=torch.int32))


# --------------------------------------------------------------------------- verification

ONE = 1 << 31


def whole(p):
    p = float(p)
    return int(min(p, 1.0) * ONE) if p > 0 else 0


def verify_ints(probs, tokens, uniforms, parents, draft):
    """One sequence, one step at a time, in Python integers."""
    T, V = len(tokens), probs.shape[1]
    us = [min(whole(u), ONE - 1) for u in uniforms]
    parents = list(range(-1, T - 1)) if parents is None else parents
    at, path = -1, []
    while True:
        p = [whole(x) for x in probs[at + 1]]
        w, left, step = list(p), ONE, None
        for c in range(at + 1, T):
            if parents[c] != at or not 0 <= tokens[c] < V:
                continue
            x = tokens[c]
            if draft is not None:
                q = [whole(y) for y in draft[c]]
                if us[c] * q[x] < p[x] * ONE:
                    step = c
                else:
                    w = [max(a - b, 0) for a, b in zip(p, q)]
            elif us[c] * max(left, 0) < w[x] * ONE:
                step = c
            else:
                left, w[x] = left - w[x], 0
            if step is not None:
                break
        if step is None:
            break
        path.append(step)
        at = step
    if not sum(w):
        w = p
    t, total, x = us[T] * sum(w) // ONE, 0, -1
    for i, y in enumerate(w):
        total += y
        if total > t:
            x = i
            break
    return path + [-1] * (T - len(path)), len(path), x


def check_verify(probs, tokens, uniforms, parents, draft):
    path, count, token = ops.verify_drafts(probs, i32(tokens), uniforms, None if parents is None else i32(parents), draft)
    p, u = probs.double().cpu().numpy(), uniforms.double().cpu().numpy()
    q = None if draft is None else draft.double().cpu().numpy()
    for b in range(len(tokens)):
        want = verify_ints(p[b], list(tokens[b]), u[b], None if parents is None else list(parents[b]), None if q is None else q[b])
        assert (path[b].tolist(), int(count[b]), int(token[b])) == want, b


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (3, 0, 50), (5, 4, 33), (2, 128, 100), (4, 9, 4999), (1, 3, 40000), (33, 2, 256)])
@pytest.mark.parametrize("mode", ["chain", "ratio", "tree"])
def test_verify(dtype, B, T, V, mode):
    g = torch.Generator(device=DEV).manual_seed(V + T)
    r = np.random.RandomState(V + T)
    logits = 2 * torch.randn(B, T + 1, V, generator=g, device=DEV)
    probs = logits.softmax(-1).to(dtype)
    uniforms = torch.rand(B, T + 1, generator=g, device=DEV)
    draft = parents = None
    tokens = probs[:, :T].float().topk(min(3, V), -1).indices.cpu().numpy()[..., 0] if T else np.zeros((B, 0), int)
    if mode == "ratio":
        draft = (logits[:, :T] + torch.randn(B, T, V, generator=g, device=DEV)).softmax(-1).to(dtype)
    if mode == "tree":
        parents = random_trees(r, B, T, 0.1) if T else np.zeros((B, 0), int)
        tokens = np.where(r.rand(B, T) < 0.7, tokens, r.randint(0, V, (B, T)))  # some brothers are alike
    check_verify(probs, tokens.tolist(), uniforms, None if parents is None else parents.tolist(), draft)


def test_verify_edges():
    """Tokens outside the vocabulary, uniform numbers of 0 and 1, rows that are zero, hold NaN,
    infinities or negative values, drafts that match the target, masses that run out."""
    nan, inf = float("nan"), float("inf")
    rows = [[0.5, 0.25, 0.25, 0.0], [nan, 1.0, nan, -1.0], [0, 0, 0, 0], [inf, 0.5, -inf, 0.25], [1.0, 0, 0, 0],
            [0.25, 0.25, 0.25, 0.25]]
    probs = torch.tensor([[rows[(b + i) % 6] for i in range(4)] for b in range(24)], device=DEV)
    tokens = [[(b + i) % 6 - 1 for i in range(3)] for b in range(24)]
    for u in (0.0, 0.2499999, 0.25, 0.5, 1.0 - 2.0 ** -24, 1.0):
        uniforms = torch.full((24, 4), u, device=DEV)
        check_verify(probs, tokens, uniforms, None, None)
        check_verify(probs, tokens, uniforms, None, probs[:, :3].contiguous())
        check_verify(probs, tokens, uniforms, None, probs[:, 1:].contiguous())
        check_verify(probs, tokens, uniforms, [[-1, -1, -1], [-1, 0, 0], [-1, 0, -2], [-2, -1, 1]] * 6, None)


def test_verify_views_and_repeats():
    """A view with padded rows, another stream, the same answer every time."""
    g = torch.Generator(device=DEV).manual_seed(0)
    probs = torch.randn(3, 5, 130, generator=g, device=DEV).softmax(-1)[..., :129]
    tokens, u = i32([[1, 2, 3, 4]] * 3), torch.rand(3, 5, generator=g, device=DEV)
    a = ops.verify_drafts(probs, tokens, u)
    b = ops.verify_drafts(probs.contiguous(), tokens, u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = ops.verify_drafts(probs, tokens, u)
    torch.cuda.synchronize()
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.parametrize("B,V", [(55, 8192), (111, 4096), (200, 2048)])
def test_verify_short_rows_over_several_blocks(B, V):
    """Rows that each block of a cluster is through with at once, so that the blocks exchange their
    sums as soon as they can; every launch gives the same."""
    g = torch.Generator(device=DEV).manual_seed(V)
    probs = torch.randn(B, 2, V, generator=g, device=DEV).softmax(-1)
    tokens = torch.randint(0, V, (B, 1), generator=g, device=DEV)
    u = torch.rand(B, 2, generator=g, device=DEV)
    check_verify(probs, tokens.tolist(), u, None, None)
    want = ops.verify_drafts(probs, tokens.int(), u)
    got = [ops.verify_drafts(probs, tokens.int(), u) for _ in range(200)]
    for out in got:
        for x, y in zip(out, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("mode", ["ratio", "tree"])
def test_verify_keeps_the_targets_distribution(mode):
    """The first token that comes out of a step (an accepted draft or the drawn one) is
    distributed as row 0, whatever was drafted: 40000 steps, each frequency within 5 standard
    deviations."""
    n, V = 40000, 6
    g = torch.Generator(device=DEV).manual_seed(1)
    p = torch.tensor([0.05, 0.4, 0.3, 0.1, 0.14, 0.01], device=DEV)
    q = torch.tensor([0.3, 0.1, 0.3, 0.2, 0.05, 0.05], device=DEV)
    u = torch.rand(n, 4, generator=g, device=DEV)
    probs = p.expand(n, 4, V).contiguous()
    if mode == "ratio":
        tokens = torch.multinomial(q, 3 * n, replacement=True, generator=g).view(n, 3).int()
        out = ops.verify_drafts(probs, tokens, u, None, q.expand(n, 3, V).contiguous())
    else:
        tokens = i32([2, 0, 4]).expand(n, 3).contiguous()
        out = ops.verify_drafts(probs, tokens, u, i32([-1, -1, -1]).expand(n, 3).contiguous())
    path, count, token = out
    first = torch.where(count > 0, tokens.gather(1, path[:, :1].clamp(min=0).long())[:, 0], token)
    freq = torch.bincount(first.long(), minlength=V).double().cpu() / n
    want = p.double().cpu()
    assert ((freq - want).abs() <= 5 * (want * (1 - want) / n).sqrt()).all()


def test_verify_refusals():
    probs = torch.full((2, 4, 8), 0.125, device=DEV)
    tokens, u = i32([[1, 2, 3]] * 2), torch.zeros(2, 4, device=DEV)
    with pytest.raises(ValueError):
        ops.verify_drafts(probs[:, :3], tokens, u)
    with pytest.raises(ValueError):
        ops.verify_drafts(probs, tokens, u[:, :3])
    with pytest.raises(ValueError):
        ops.verify_drafts(probs, tokens, u.double())
    with pytest.raises(TypeError):
        ops.verify_drafts(probs, tokens.long(), u)
    with pytest.raises(TypeError):
        ops.verify_drafts(probs.half(), tokens, u)
    with pytest.raises(ValueError, match="chain"):
        ops.verify_drafts(probs, tokens, u, tokens, probs[:, :3])
    with pytest.raises(ValueError):
        ops.verify_drafts(probs, tokens, u, None, probs[:, :3].to(BF))
    with pytest.raises(ValueError, match="129"):
        ops.verify_drafts(torch.zeros(1, 130, 8, device=DEV), torch.zeros(1, 129, dtype=torch.int32, device=DEV),
                          torch.zeros(1, 130, device=DEV))
