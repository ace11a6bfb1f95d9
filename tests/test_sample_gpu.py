"""Sampling against a plain statement of it in whole numbers on the host, at the sizes and values where
it can go wrong."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nkilab import _native as N
from nkilab import ops

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
DEV = "cuda"
ONE = 1 << 31


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def f32(x):
    return torch.tensor(x, dtype=torch.float32, device=DEV)


def reference(row, u, t=1.0, k=0, p=1.0, low=0.0):
    """(token, prob, how far the drawn place is from its ends, as a part of the sum)."""
    x = np.where(np.isnan(row), -np.inf, row.astype(np.float64)) + 0.0
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    if not len(order):
        return -1, 0.0, 1.0
    if not t > 0:
        return int(order[0]), 1.0, 1.0
    if k > 0:
        order = order[:k]
    with np.errstate(invalid="ignore"):
        z = np.where(x[order] == x[order[0]], 0.0, (x[order] - x[order[0]]) / t)
    w = np.floor(np.exp(z) * ONE).astype(np.int64)
    if p < 1:
        need = max(1, int(w.sum()) * int(max(p, 0.0) * ONE) // ONE)
        n = int((np.cumsum(w) < need).sum()) + 1
        order, w = order[:n], w[:n]
    if low > 0:
        n = int((w >= min(low, 1.0) * ONE).sum())
        order, w = order[:n], w[:n]
    back = np.argsort(order)
    sums = np.cumsum(w[back])
    total = int(sums[-1])
    place = total * min(int(u * ONE), ONE - 1) // ONE
    at = int((sums <= place).sum())
    return int(order[back[at]]), float(w[back[at]]) / total, min(int(sums[at]) - place, place - int(sums[at]) + int(w[back[at]])) / total


def check(logits, u, got, **kw):
    """Weights are equal to the reference's but for a unit in the last place now and then, where the product
    with 2^31 is within rounding of a whole number: some 1e-9 of the sum, which decides a draw only
    at a place that near to a border."""
    token, prob = got
    assert token.dtype == torch.int32 and prob.dtype == torch.float32
    rows, us = logits.float().cpu().numpy(), u.double().cpu().numpy()
    for b in range(len(us)):
        own = {n: float(v[b] if torch.is_tensor(v) else np.float32(v)) for n, v in kw.items()}
        if "k" in own:
            own["k"] = int(own["k"])
        want, share, near = reference(rows[b], us[b], **own)
        if near > 1e-8:
            assert int(token[b]) == want, (b, own)
            assert abs(float(prob[b]) - share) <= 2.0 ** -23 * share + 2.0 ** -31 / max(share, 1e-9) * 1e-6 + 1e-9


FILTERS = [dict(), dict(t=0.7), dict(t=2.5, k=40), dict(p=0.9), dict(t=0.8, p=0.95, k=500), dict(low=0.05),
           dict(t=1.3, p=0.5, low=0.001), dict(t=0.0), dict(k=1), dict(p=0.0), dict(low=1.0), dict(k=3, p=0.6, low=0.2, t=5.0),
           dict(k=10 ** 9), dict(t=1e-30), dict(t=1e30, p=0.3)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,V", [(3, 1), (5, 2), (2, 31), (4, 1000), (1, 4097), (2, 32768), (3, 50257), (40, 9001), (1, 131072), (2, 262147)])
def test_sample(B, V, dtype):
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = (torch.randn(B, V, generator=g, device=DEV) * 3).to(dtype)
    for i, kw in enumerate(FILTERS):
        u = torch.rand(B, generator=g, device=DEV)
        if i == 0:
            u[0] = 0.0
            u[-1] = 1.0 - 2.0 ** -24
        got = ops.sample(logits, u, kw.get("t", 1.0), kw.get("k", 0), kw.get("p", 1.0), kw.get("low", 0.0))
        check(logits, u, got, **kw)


def test_the_largest_vocabulary():
    logits = torch.randn(2, N.MAX_VOCAB, device=DEV) * 2
    u = torch.rand(2, device=DEV)
    check(logits, u, ops.sample(logits, u, 0.9, 2000, 0.9), t=0.9, k=2000, p=0.9)


@pytest.mark.parametrize("V", [700, 40000])
def test_settings_of_each_row(V):
    r = np.random.RandomState(V)
    B = 64
    logits = torch.randn(B, V, device=DEV) * 2.5
    u = torch.rand(B, device=DEV)
    t, k = f32(r.choice([0.0, 0.5, 1.0, -1.0, float("nan"), 2.0], B).tolist()), i32(r.choice([0, 1, 2, 50, -3, 10 ** 6], B).tolist())
    p, low = f32(r.choice([1.0, 0.9, 0.1, float("nan"), 2.0, -1.0], B).tolist()), f32(r.choice([0.0, 0.1, float("nan"), 7.0], B, p=[0.5, 0.2, 0.2, 0.1]).tolist())
    got = ops.sample(logits, u, t, k, p, low)
    own = dict(t=torch.nan_to_num(t, 0.0), k=k.clamp_min(0), p=torch.nan_to_num(p, 1.0), low=torch.nan_to_num(low, 0.0))
    check(logits, u, got, **own)
    for b in (0, 7, 33):  # one by one
        one = ops.sample(logits[b:b + 1], u[b:b + 1], t[b:b + 1], k[b:b + 1], p[b:b + 1], low[b:b + 1])
        assert int(one[0]) == int(got[0][b]) and float(one[1]) == float(got[1][b])


@pytest.mark.parametrize("V", [100, 5000, 70000])
def test_ties(V):
    """Rows of few different values: of equal ones the lowest index stays."""
    r = np.random.RandomState(V)
    rows = [np.zeros(V), np.full(V, -7.5), r.randint(0, 2, V) * 1.0, r.randint(-3, 4, V) * 0.25, np.where(r.rand(V) < 0.01, 0.0, -np.inf),
            np.where(np.arange(V) % 2 == 0, 0.0, -0.0), np.where(np.arange(V) == V - 1, 3.0, 2.0)]
    logits = f32(np.stack(rows).tolist())
    for kw in (dict(), dict(k=7), dict(p=0.3), dict(k=V // 2 + 1, p=0.7), dict(low=0.9), dict(k=V - 1, t=0.3), dict(p=0.999)):
        for _ in range(2):
            u = torch.rand(len(rows), device=DEV)
            check(logits, u, ops.sample(logits, u, kw.get("t", 1.0), kw.get("k", 0), kw.get("p", 1.0), kw.get("low", 0.0)), **kw)


@pytest.mark.parametrize("V", [8, 3000, 33000])
def test_values(V):
    inf, nan = float("inf"), float("nan")
    r = np.random.RandomState(V)
    rows = np.tile(r.randn(V) * 2, (12, 1))
    rows[0] = -inf
    rows[1] = nan
    rows[2, :] = -inf
    rows[2, V // 2] = -1000.0
    rows[3, 1::2] = nan
    rows[4, [0, V - 1]] = inf
    rows[5, ::3] = -inf
    rows[6] = np.where(np.arange(V) % 2, 3.4e38, -3.4e38)
    rows[7] *= 1e-42
    rows[8] = -rows[8] * 1e30
    rows[9] = 1e-45 * np.arange(V)
    rows[10] = np.linspace(-60, 0, V)
    rows[11, 5:] = -80.0
    logits = torch.tensor(rows, dtype=torch.float32, device=DEV)
    for kw in (dict(), dict(p=0.9), dict(k=5), dict(k=9, p=0.99, low=1e-6), dict(t=30.0, p=0.8), dict(t=0.01, k=3), dict(t=0.0)):
        u = torch.rand(12, device=DEV)
        check(logits, u, ops.sample(logits, u, kw.get("t", 1.0), kw.get("k", 0), kw.get("p", 1.0), kw.get("low", 0.0)), **kw)
    got = ops.sample(logits[:2], f32([nan, 5.0]))
    assert got[0].tolist() == [-1, -1] and got[1].tolist() == [0.0, 0.0]
    got = ops.sample(logits[10:11].expand(4, V), f32([nan, -1.0, 1.0, inf]))  # taken as 0, 0 and the last place
    assert int(got[0][0]) == int(got[0][1]) and int(got[0][2]) == int(got[0][3])


def test_a_grid_of_uniform_numbers_gives_the_distribution():
    """Numbers spread evenly meet each token as often as its probability says, to one."""
    V, B = 37, 4096
    logits = torch.randn(1, V, device=DEV, dtype=F32)
    u = (torch.arange(B, device=DEV, dtype=F32) + 0.5) / B
    for kw in (dict(), dict(k=10), dict(p=0.8), dict(low=0.2)):
        token, prob = ops.sample(logits.expand(B, V), u, 0.9, kw.get("k", 0), kw.get("p", 1.0), kw.get("low", 0.0))
        p = torch.softmax(logits.double()[0] / 0.9, 0)
        counts = torch.bincount(token.long(), minlength=V).double()
        kept = counts > 0
        share = p * kept / (p * kept).sum()
        assert (counts - share * B).abs().max() < 1.5
        assert (prob.double() - share[token.long()]).abs().max() < 1e-6
        assert torch.equal(token.sort().values, token)  # by index


def test_layouts_repeats_streams_and_graphs():
    g = torch.Generator(device=DEV).manual_seed(1)
    wide = torch.randn(6, 3, 30011, generator=g, device=DEV)
    logits, u = wide[:, 1], torch.rand(6, generator=g, device=DEV)
    want = ops.sample(logits, u, 0.8, 100, 0.9)
    check(logits, u, want, t=0.8, k=100, p=0.9)
    for x in (logits.contiguous(), logits.mT.contiguous().mT, torch.zeros(6 * 30011 + 1, device=DEV)[1:].view(6, -1).copy_(logits)):
        got = ops.sample(x, u, 0.8, 100, 0.9)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for s in (side, other):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            assert torch.equal(ops.sample(logits, u, 0.8, 100, 0.9)[0], want[0])
            graph = torch.cuda.CUDAGraph()
            s.synchronize()
            with torch.cuda.graph(graph, stream=s):
                out = ops.sample(logits, u, 0.8, 100, 0.9)
            graphs.append((s, graph, out))
    for s, graph, _ in graphs * 3:
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for _, _, out in graphs:
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_past_32_bits():
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    big = torch.empty(22000, 131072, dtype=BF, device=DEV)  # 2.9e9 values
    big[-3:].normal_()
    u = torch.rand(3, device=DEV)
    want = ops.sample(big[-3:].clone(), u, 1.0, 0, 0.9)
    big[:-3].fill_(1.0)
    token, prob = ops.sample(big, torch.cat([torch.full((21997,), 0.25, device=DEV), u]), 1.0, 0, 0.9)
    assert torch.equal(token[-3:], want[0]) and torch.equal(prob[-3:], want[1])
    assert (token[:-3] == token[0]).all()


def test_refusals_and_nothing_to_do():
    x, u = torch.randn(2, 10, device=DEV), torch.rand(2, device=DEV)
    for bad in (lambda: ops.sample(x[0], u), lambda: ops.sample(x, u[:1]), lambda: ops.sample(x[:, :0], u), lambda: ops.sample(x, u, -1.0),
                lambda: ops.sample(x, u, float("nan")), lambda: ops.sample(x, u, 1.0, -1), lambda: ops.sample(x, u, top_p=1.5),
                lambda: ops.sample(x, u, min_p=-0.1), lambda: ops.sample(x, u, u[:1]), lambda: ops.sample(x, u, top_k=i32([1]))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.sample(x.half(), u), lambda: ops.sample(x, u.double()), lambda: ops.sample(x, u, top_k=u), lambda: ops.sample(x, u, u.double())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(N.NklError):
        ops.sample(torch.zeros(1, N.MAX_VOCAB + 1, device=DEV), u[:1])
    with pytest.raises(RuntimeError):
        ops.sample(x, u.cpu())
    assert ops.sample(x[:0], u[:0])[0].shape == (0,)
    token, prob = ops.sample(x.clone().requires_grad_(), u)
    with pytest.raises(RuntimeError, match="sample"):
        prob.sum().backward()
