"""Attention over a cache in 8 bits against a plain statement of it in 64 bits, at the sizes, masks
and values where it can go wrong."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from nkilab import _native as N
from nkilab import ops
from test_decode_gpu import ATTENTION, attention_64, i32, random_trees

pytestmark = pytest.mark.gpu

BF, F32, E4M3, E8M0 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float8_e8m0fnu
DEV = "cuda"


def values(cache, scales):
    return (cache.float().unflatten(-2, (scales.shape[-1], -1)) * scales.float()[..., None, None]).flatten(-3, -2)


def setup(B, T, H, Hkv, d, page, block, lens, dtype, seed=0, layout="heads", spare=3, spread=3):
    """Inputs whose cache holds bytes of all kinds wherever no sequence looks."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = np.random.RandomState(seed)
    M = max(1, max(-(-n // page) for n in lens)) + 1
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    order, at = r.permutation(P), 0
    shape = (P, Hkv, page, d) if layout == "heads" else (P, page, Hkv, d)
    kc, vc = (torch.randint(0, 256, shape, generator=g, device=DEV).to(torch.uint8).view(E4M3) for _ in range(2))
    if layout != "heads":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    ks, vs = (torch.randint(0, 256, (P, Hkv, page // block), generator=g, device=DEV).to(torch.uint8).view(E8M0) for _ in range(2))
    tables = np.full((B, M), -1)
    for b, n in enumerate(lens):
        tables[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    tables = i32(tables.tolist())
    most = max(lens)
    if most:  # rows whose blocks differ in size
        rows = [torch.randn(1, B, most, Hkv, d, generator=g, device=DEV) for _ in range(2)]
        for x in rows:
            x *= torch.exp2(torch.randint(-spread, spread + 1, (1, B, -(-most // block), Hkv, 1), generator=g, device=DEV).float()).repeat_interleave(block, 2)[:, :, :most]
        rows[0] *= 0.3
        ops.cache_append(*rows, kc[None], vc[None], tables, i32([0] * B), None, i32(lens), ks[None], vs[None])
    q, k, v = torch.randn(B, T, H + 2 * Hkv, d, generator=g, device=DEV).to(dtype).split([H, Hkv, Hkv], 2)
    return q, k, v, kc, vc, tables, i32(lens), ks, vs


def check(got, want, mag, dtype, on_tcgen05=False):
    """Scores: sums of up to 128 products in fp32, and the exponentials, each within some 2^-24 of their
    sizes: as 2e-5 (1 + sum p |v|) for the older kernels. bf16: the output's rounding, half a step, and
    that of the weights, half a step each, of f16 or, on tcgen05 (more than 16 rows to a key/value head), of
    bf16; 5 % for the products of the two."""
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    bound = 2e-5 * (1 + mag)
    if dtype == BF:
        bound = bound + 2.0 ** -8 * want.abs() + 1.05 * (2.0 ** -8 if on_tcgen05 else 2.0 ** -11) * mag
    err = (got - want).abs()
    assert (err <= bound).all(), float((err / bound).max())


def run(x, parents=None, scale=None):
    q, k, v, kc, vc, tables, lens, ks, vs = x
    return ops.attention_tree(q, k, v, kc, vc, tables, lens, parents, scale, ks, vs)


def exact(x, parents=None, scale=None):
    q, k, v, kc, vc, tables, lens, ks, vs = x
    return attention_64(q, k, v, values(kc, ks), values(vc, vs), tables, lens, parents, scale or 1 / math.sqrt(q.shape[-1]))


def block_of(page, at):
    blocks = [b for b in (page, 16, 8, 4, 1) if page % b == 0]
    return blocks[at % min(3, len(blocks))]


CASES = [c for c in ATTENTION if c[4] % 16 == 0] + [
    (2, 1, 4, 4, 16, 16, [40, 5], BF),
    (3, 4, 6, 2, 48, 32, [500, 31, 0], F32),
    (2, 9, 4, 1, 112, 48, [333, 96], BF),
    (1, 1, 64, 1, 80, 64, [1500], F32),       # 64 heads share
    (2, 128, 8, 8, 32, 16, [17, 260], F32),
    (6, 1, 16, 2, 128, 64, [5000, 3, 64, 32, 31, 33], BF),
]


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("at", range(len(CASES)))
def test_attention_8bit(at, tree):
    B, T, H, Hkv, d, page, lens, dtype = CASES[at]
    x = setup(B, T, H, Hkv, d, page, block_of(page, at + tree), lens, dtype, seed=at)
    parents = i32(random_trees(np.random.RandomState(at), B, T).tolist()) if tree else None
    check(run(x, parents), *exact(x, parents), dtype, T * H // Hkv > 16 and d in (64, 128) and page % 8 == 0)


@pytest.mark.parametrize("T,H,Hkv,d,page,lens", [(33, 4, 4, 128, 64, [700, 0, 63]), (16, 8, 2, 64, 24, [1000, 128]), (128, 4, 1, 128, 16, [900, 40]),
                                                 (20, 12, 4, 64, 256, [127, 129, 2500]), (64, 32, 8, 128, 32, [3000, 5])])
def test_many_rows_equal_the_bf16_cache(T, H, Hkv, d, page, lens):
    """On tcgen05 the cache's values become bf16 without a rounding: the same bits as over a cache that holds them in bf16."""
    x = setup(len(lens), T, H, Hkv, d, page, 8, lens, BF, seed=T)
    parents = i32(random_trees(np.random.RandomState(T), len(lens), T).tolist())
    q, k, v, kc, vc, tables, n, ks, vs = x
    kc, vc = (torch.nan_to_num(values(c, s), 0.0, 1e30, -1e30).to(BF) for c, s in ((kc, ks), (vc, vs)))
    assert torch.equal(run(x, parents), ops.attention_tree(q, k, v, kc, vc, tables, n, parents))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_layouts(dtype):
    x = setup(3, 5, 8, 2, 64, 16, 8, [100, 0, 37], dtype, layout="rows")
    check(run(x), *exact(x), dtype)
    q, k, v = x[:3]
    want = run(x)
    assert torch.equal(run((q.contiguous(), k.contiguous(), v.contiguous(), *x[3:])), want)
    dense = [c.contiguous() for c in x[3:5]]
    assert torch.equal(run((q, k, v, *dense, *x[5:])), want)
    odd = [torch.zeros(t.numel() + 1, device=DEV, dtype=dtype)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert torch.equal(run((*odd, *x[3:])), want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 128])
def test_scores_of_all_sizes(dtype, d):
    """Scales that are negative, large scores, queries of very different sizes, growing maxima."""
    x = list(setup(2, 4, 8, 2, d, 32, 16, [700, 90], dtype, seed=5))
    for scale in (-0.2, 3.0, 1e-8, 0.0):
        want, mag = exact(x, None, scale or 1e-300)
        check(run(x, None, scale), want, mag * (1 + 200 * abs(scale)), dtype)  # a score of some 200 is off by 200 * 2^-22 or so
    x[0] = x[0] * torch.exp2(torch.randint(-60, -20, (2, 4, 8, 1), device=DEV).to(dtype))
    check(run(x), *exact(x), dtype)
    x[0] = x[0] * 2.0 ** 40
    q = torch.zeros_like(x[0])
    q[..., 0] = 8
    x[0] = q
    k = values(x[3], x[7])
    k[..., 0] = torch.linspace(-30, 30, k.shape[0] * k.shape[2], device=DEV).view(k.shape[0], 1, k.shape[2])
    rows = k[x[5][:, :22].clamp_min(0).long()].transpose(2, 3).flatten(1, 2)[None, :, :700]  # in order of position
    rows[0, :, :, :, 0] = torch.linspace(-30, 30, 700, device=DEV)[:, None]
    ops.cache_append(rows, rows.flip(2) * 0.01, x[3][None], x[4][None], x[5], i32([0, 0]), None, x[6], x[7][None], x[8][None])
    want, mag = exact(x)
    check(run(x), want, 20 * mag, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_powers_far_apart(dtype):
    """Blocks whose powers of two differ by 2^40, the smallest and the largest: weights for v have a
    maximum of their own."""
    x = list(setup(1, 2, 4, 2, 64, 64, 16, [300], dtype, seed=2, spread=0))
    rows = [torch.randn(1, 1, 300, 2, 64, device=DEV) for _ in range(2)]
    size = torch.exp2(20.0 * torch.randint(-1, 2, (19,), device=DEV)).repeat_interleave(16)[:300, None, None]
    append = lambda k, v: ops.cache_append(k, v, x[3][None], x[4][None], x[5], i32([0]), None, None, x[7][None], x[8][None])  # noqa: E731
    for v in (rows[1] * size, rows[1] * size.flip(0), rows[1] * 2.0 ** -90, rows[1] * 2.0 ** 100, rows[1] * size * 2.0 ** 30):
        append(rows[0], v)
        want, mag = exact(x)
        got = run(x).double().cpu()
        bound = 4e-5 * mag + (2.0 ** -8 * want.abs() + 1.05 * 2.0 ** -11 * mag if dtype == BF else 0) + 2e-5 * x[2].double().abs().max().item()
        assert ((got - want).abs() <= bound).all()
    # the keys of one block weigh 2^-24 and less, their v is 2^30 times the others'
    q = torch.zeros_like(x[0])
    q[..., 0] = 8.0
    k = torch.zeros_like(rows[0])
    k[0, 0, 32:48, :, 0] = -20.0
    v = rows[1].clone()
    v[0, 0, 32:48] *= 2.0 ** 30
    append(k, v)
    y = [q, torch.zeros_like(x[1]), x[2], *x[3:]]
    want, mag = exact(y)
    got = run(y).double().cpu()
    assert ((got - want).abs() <= 6e-5 * mag + 2.0 ** -8 * want.abs() + 1.05 * 2.0 ** -11 * mag).all()


@pytest.mark.parametrize("dtype,d,page,T", [(BF, 128, 64, 2), (BF, 64, 24, 3), (F32, 64, 16, 2), (F32, 96, 8, 20), (BF, 128, 16, 12), (BF, 64, 32, 60)])
def test_infinities_and_nan(dtype, d, page, T):
    """Of tokens and blocks that a row sees they show, of the others not."""
    lens = [70, 130]
    base = setup(2, T, 4, 2, d, page, 8, lens, dtype, seed=3)
    parents = i32([[-1] * T, [-1] * T])  # each sees the cache and itself
    want = run(base, parents)
    junk = float("nan")
    for name, value in ((1, junk), (2, junk), (1, float("inf")), (2, float("inf")), (2, float("-inf")), (0, junk)):
        x = [t.clone() if i < 3 else t for i, t in enumerate(base)]
        x[name][0, 1, 0, 5] = value
        got = run(x, parents)
        hit = torch.zeros_like(want, dtype=torch.bool)
        heads = slice(0, 2) if name else slice(0, 1)
        if name == 2:
            hit[0, 1, heads, 5] = True
            assert (got[0, 1, heads, 5] == value).all() or math.isnan(value) and got[0, 1, heads, 5].isnan().all()
        elif value != value:
            hit[0, 1, heads] = True
            assert got[0, 1, heads].isnan().all()
        else:  # a key of infinity: the scores are infinities of either sign
            ref = attention_64(x[0], x[1], x[2], values(x[3], x[7]), values(x[4], x[8]), *x[5:7], parents, 1 / math.sqrt(d))[0]
            hit[0, 1, heads] = True
            assert torch.equal(got[0, 1, heads].isnan().cpu(), ref[0, 1, heads].isnan())
            fine = ~ref[0, 1, heads].isnan()
            assert (got[0, 1, heads].double().cpu()[fine] - ref[0, 1, heads][fine]).abs().max() < 0.05 if fine.any() else True
        assert torch.equal(got[~hit], want[~hit])
        gone = parents.clone()
        gone[0, 1] = -2  # an absent token: zeros, and nothing of it anywhere
        got = run(x, gone)
        assert not got[0, 1].any() and torch.equal(got[0, 0], want[0, 0]) and torch.equal(got[1], want[1])
    # a block of the cache that is NaN
    x = list(base)
    for which in (7, 8):
        x[which] = base[which].clone()
        p = int(base[5][0, 0])
        x[which].view(torch.uint8)[p, 1, 0] = 255
        got = run(x, parents)
        assert got[0, :, 2:].isnan().all() and torch.equal(got[0, :, :2], want[0, :, :2]) and torch.equal(got[1], want[1])
        x[which] = base[which]


def test_tables_out_of_range_are_harmless():
    x = list(setup(2, 2, 4, 2, 64, 16, 16, [100, 60], BF))
    want = run(x)
    x[5] = x[5].clone()
    x[5][1] = i32([1 << 30, -7, 9999, 14, -1, -1, -1, -1][:x[5].shape[1]])
    got = run(x)
    assert torch.equal(got[0], want[0]) and torch.isfinite(got[1]).all()
    for lens in ([-5, 1 << 30], [0, 0]):
        x[6] = i32(lens)
        assert torch.isfinite(run(x)[0]).all()


@pytest.mark.parametrize("dtype,T", [(BF, 1), (BF, 40), (F32, 3)])
def test_repeats_streams_and_graphs(dtype, T):
    x = setup(3, T, 8, 2, 128, 64, 16, [3000, 100, 2000], dtype)
    want = run(x)
    assert torch.equal(run(x), want)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for s in (side, other):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            assert torch.equal(run(x), want)
            graph = torch.cuda.CUDAGraph()
            s.synchronize()
            with torch.cuda.graph(graph, stream=s):
                out = run(x)
            graphs.append((graph, out))
    for _ in range(3):
        for s, (graph, _) in zip((side, other), graphs):  # two graphs at once: workspaces of their own
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert torch.equal(out, want)


def test_past_32_bits():
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB")
    for layout in ("heads", "rows"):
        P = (1 << 32) // (4 * 64 * 128) + 9
        shape = (P, 4, 64, 128) if layout == "heads" else (P, 64, 4, 128)
        kc, vc = (torch.zeros(shape, device=DEV, dtype=torch.uint8).view(E4M3) for _ in range(2))
        if layout == "rows":
            kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
        ks, vs = (torch.full((P, 4, 4), 127, device=DEV, dtype=torch.uint8).view(E8M0) for _ in range(2))
        rows = [torch.randn(1, 1, 150, 4, 128, device=DEV) for _ in range(2)]
        tables = i32([[P - 1, P - 3, P - 8]])
        ops.cache_append(*rows, kc[None], vc[None], tables, i32([0]), None, None, ks[None], vs[None])
        q, k, v = (torch.randn(1, 3, h, 128, device=DEV).to(BF) for h in (8, 4, 4))
        got = ops.attention_tree(q, k, v, kc, vc, tables, i32([150]), k_scales=ks, v_scales=vs)
        few = [t[[P - 1, P - 3, P - 8]].contiguous() for t in (kc, vc)]
        small = [t[[P - 1, P - 3, P - 8]].contiguous() for t in (ks, vs)]
        assert torch.equal(got, ops.attention_tree(q, k, v, *few, i32([[0, 1, 2]]), i32([150]), k_scales=small[0], v_scales=small[1]))
        del kc, vc


def test_refusals_and_nothing_to_do():
    x = setup(2, 3, 4, 2, 64, 16, 8, [20, 5], BF)
    q, k, v, kc, vc, tables, lens, ks, vs = x
    call = ops.attention_tree
    for bad in ((q, k, v, kc, vc, tables, lens, None, None, ks), (q, k, v, kc, vc, tables, lens, None, None, ks[:1], vs),
                (q[:, :, :3], k, v, kc, vc, tables, lens, None, None, ks, vs), (q, k[:1], v, kc, vc, tables, lens, None, None, ks, vs),
                (q, k, v, kc, vc, tables[0], lens, None, None, ks, vs), (q, k, v, kc[None], vc[None], tables, lens, None, None, ks, vs)):
        with pytest.raises(ValueError):
            call(*bad)
    for bad in ((q, k, v, kc.float(), vc.float(), tables, lens, None, None, ks, vs), (q, k.float(), v, kc, vc, tables, lens, None, None, ks, vs),
                (q, k, v, kc, vc, tables, lens, None, None, ks.float(), vs.float()), (q.half(), k.half(), v.half(), kc, vc, tables, lens, None, None, ks, vs),
                (q, k, v, kc, vc, tables, lens)):
        with pytest.raises(TypeError):
            call(*bad)
    with pytest.raises(RuntimeError):
        call(q, k, v, kc, vc, tables, lens.cpu(), None, None, ks, vs)
    with pytest.raises(ValueError):
        call(q.new_zeros(2, 129, 4, 64), k.new_zeros(2, 129, 2, 64), k.new_zeros(2, 129, 2, 64), kc, vc, tables, lens, None, None, ks, vs)
    with pytest.raises(N.NklError):  # 24 entries
        c = torch.zeros(4, 2, 16, 24, device=DEV).to(E4M3)
        call(q[..., :24], k[..., :24], v[..., :24], c, c, tables, lens, None, None, ks[:4], vs[:4])
    out = call(q.clone().requires_grad_(), k, v, kc, vc, tables, lens, None, None, ks, vs)
    with pytest.raises(RuntimeError, match="attention_tree_8bit"):
        out.sum().backward()
    assert call(q[:, :0], k[:, :0], v[:, :0], kc, vc, tables, lens, None, None, ks, vs).shape == (2, 0, 4, 64)
    assert call(q[:0], k[:0], v[:0], kc, vc, tables[:0], lens[:0], None, None, ks, vs).shape == (0, 3, 4, 64)
