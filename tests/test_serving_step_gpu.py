"""nkilab.serving with rotary positions, 8-bit caches and sampling: the operators together, as a decoding
loop uses them."""
from __future__ import annotations

import math

import pytest
import torch

from nkilab import ops
from nkilab.model import BlockConfig, DecoderBlock
from nkilab.serving import PagedCache, Rotary, decode, extend, next_token, speculative_step, step

pytestmark = pytest.mark.gpu
DEV, BF, F32, E4M3 = "cuda", torch.bfloat16, torch.float32, torch.float8_e4m3fn


def blocks_of(layers, d_model=256, heads=4, d_ff=384):
    torch.manual_seed(3)
    return [DecoderBlock(BlockConfig(d_model, heads, d_ff)).to(DEV).eval() for _ in range(layers)]


def whole(blocks, x, rotary):
    """The blocks with rotary positions in 64 bits, x [S, d]."""
    x = x.double()
    f = rotary.freqs
    n = f.numel()
    angle = torch.arange(len(x), device=DEV).double()[:, None, None] * f
    c, s = angle.cos() * rotary.magnitude, angle.sin() * rotary.magnitude

    def turn(t):
        i, j = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if rotary.interleaved else (slice(0, n), slice(n, 2 * n))
        y = t.clone()
        y[..., i], y[..., j] = t[..., i] * c - t[..., j] * s, t[..., j] * c + t[..., i] * s
        return y

    norm = lambda t, m: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + m.eps) * m.weight.double()  # noqa: E731
    for b in blocks:
        H, hd = b.cfg.n_heads, b.cfg.head_dim
        q, k, v = (norm(x, b.norm1) @ b.wqkv.weight.double().T).view(len(x), 3, H, hd).unbind(1)
        q, k = turn(q), turn(k)
        w = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(hd)
        w = w.masked_fill(torch.ones_like(w[0]).triu(1).bool(), -math.inf).softmax(-1)
        x = x + torch.einsum("hij,jhd->ihd", w, v).reshape(len(x), -1) @ b.wo.weight.double().T
        h = norm(x, b.norm2)
        x = x + (torch.nn.functional.silu(h @ b.wg.weight.double().T) * (h @ b.wu.weight.double().T)) @ b.wd.weight.double().T
    return x


# fp32: some hundred roundings of 2^-24 through two layers; bf16: 2^-8 for each of some 20 roundings on the way, of
# which a residual keeps a part
BOUND = {F32: 2e-4, BF: 6e-2}


@pytest.mark.parametrize("dtype,interleaved,part", [(F32, False, 64), (F32, True, 32), (BF, False, 64)])
def test_prompts_and_tokens_equal_the_whole(dtype, interleaved, part):
    """A padded batch of prompts longer than a chunk, then single tokens, then a tree's first path."""
    blocks, rotary = blocks_of(2), Rotary(64, part, scaling="yarn", factor=4.0, trained=64, interleaved=interleaved)
    S, n = 170, [150, 133]
    x = torch.randn(2, S, 256, device=DEV).to(dtype)
    want = [whole(blocks, x[b], rotary) for b in range(2)]
    cache = PagedCache(2, 2, 30, 4, 64, page_size=16, dtype=dtype)
    cache.reserve(S)
    close = lambda got, ref: (got.double() - ref).abs().max() / ref.abs().max() < BOUND[dtype]  # noqa: E731
    y = extend(blocks, x[:, :150], cache, rotary, torch.tensor(n, dtype=torch.int32, device=DEV))
    assert cache.lens.tolist() == n
    for b in range(2):
        assert close(y[b, :n[b]], want[b][:n[b]])
    for t in range(3):
        now = torch.stack([x[b, n[b] + t] for b in range(2)])[:, None]
        y = extend(blocks, now, cache, rotary)
        for b in range(2):
            assert close(y[b, 0], want[b][n[b] + t])
    now = torch.stack([x[b, n[b] + 3:n[b] + 7] for b in range(2)])
    tree = torch.cat([now[:, :2], torch.randn_like(now[:, :1]), now[:, 2:]], 1)
    parents = torch.tensor([[-1, 0, 0, 1, 3]] * 2, dtype=torch.int32, device=DEV)
    y, k, v = decode(blocks, tree, cache, parents, rotary)
    for b in range(2):
        assert close(y[b, [0, 1, 3, 4]], want[b][n[b] + 3:n[b] + 7])
    path = torch.tensor([[0, 1, 3, 4, -1]] * 2, dtype=torch.int32, device=DEV)
    cache.append(k, v, path, torch.full_like(cache.lens, 4))
    y = extend(blocks, torch.stack([x[b, n[b] + 7] for b in range(2)])[:, None], cache, rotary)
    for b in range(2):
        assert close(y[b, 0], want[b][n[b] + 7])


@pytest.mark.parametrize("dtype", [BF, F32, E4M3])
def test_steps_are_their_operators(dtype):
    """A step gives, bit for bit, what its operators give one by one."""
    rows = F32 if dtype == F32 else BF
    blocks, rotary, V, B = blocks_of(2), Rotary(64), 96, 3
    g = torch.Generator(device=DEV).manual_seed(5)
    embedding = torch.randn(V, 256, generator=g, device=DEV).to(rows)
    head = (torch.randn(256, V, generator=g, device=DEV) * 0.2).to(rows)
    a, b = (PagedCache(2, B, 30, 4, 64, page_size=16, dtype=dtype, block=8) for _ in range(2))
    prompt = embedding[torch.randint(0, V, (B, 40), generator=g, device=DEV)]
    for c in (a, b):
        for t in (c.k, c.v):  # rows that nothing writes are equal too
            t.view(torch.uint8).zero_()
        c.reserve(60)
    # prompts: rotated and appended in one pass, or one by one
    extend(blocks, prompt, a, rotary)
    y, k, v = decode(blocks, prompt, b, None, rotary)
    if dtype != E4M3:  # there the one pass rounds once
        b.append(k, v)
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    b.k.copy_(a.k), b.v.copy_(a.v), b.lens.copy_(a.lens)
    if dtype == E4M3:
        b.k_scales.copy_(a.k_scales), b.v_scales.copy_(a.v_scales)
    last = torch.tensor([3, 90, 17], dtype=torch.int32, device=DEV)
    for i in range(4):
        u = torch.rand(B, generator=g, device=DEV)
        token, prob = step(blocks, embedding, head, a, last, u, rotary, 0.8, 20, 0.9, 0.01)
        x = embedding[last.long()][:, None]
        y, k, v = decode(blocks, x, b, None, rotary)
        want = next_token(y[:, 0], head, u, 0.8, 20, 0.9, 0.01)
        assert torch.equal(token, want[0]) and torch.equal(prob, want[1])
        b.append(k, v)
        assert torch.equal(a.lens, b.lens) and a.lens.tolist() == [41 + i] * B
        if dtype == E4M3:
            b.k.copy_(a.k), b.k_scales.copy_(a.k_scales)
            assert torch.equal(a.v_scales.view(torch.uint8), b.v_scales.view(torch.uint8))
        assert torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8)) and torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8))
        last = token


def values(cache, slot):
    """A slot's k and v in 32 bits, [2, layers, heads, positions, head_dim]."""
    n = int(cache.lens[slot])
    pages = cache.tables[slot, :-(-n // cache.page_size)].long()
    out = []
    for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        x = c[:, pages].float().unflatten(3, (s.shape[-1], -1)) * s[:, pages].float()[..., None, None]
        out.append(x.flatten(3, 4).transpose(1, 2).flatten(2, 3)[:, :, :n])
    return torch.stack(out)


def test_forks_and_compaction_take_the_scales_along():
    cache = PagedCache(2, 5, 40, 3, 32, page_size=16, dtype=E4M3, block=4, max_len=80)
    g = torch.Generator(device=DEV).manual_seed(1)

    def grow(n):
        T = max(n)
        cache.reserve(torch.tensor(n, dtype=torch.int32))
        rows = [torch.randn(2, 5, T, 3, 32, generator=g, device=DEV) * torch.exp2(torch.randint(-9, 9, (2, 5, T, 3, 1), generator=g, device=DEV).float()) for _ in range(2)]
        path = torch.arange(T, dtype=torch.int32, device=DEV).expand(5, T).contiguous()
        cache.append(*rows, path, torch.tensor(n, dtype=torch.int32, device=DEV))

    grow([21, 32, 7, 0, 50])
    was = [values(cache, s) for s in range(5)]
    # onto itself, out of range, twice into the same slot: skipped
    assert cache.fork([0, 4, 1, 9, 0, 2], [3, 2, 1, 0, 2, -1]).item() == 0
    assert cache.lens.tolist() == [21, 32, 50, 21, 50]
    for slot, src in ((0, 0), (1, 1), (2, 4), (3, 0), (4, 4)):
        assert torch.equal(values(cache, slot), was[src])
    grow([3, 1, 2, 9, 0])
    now = [values(cache, s) for s in range(5)]
    assert torch.equal(now[3][:, :, :, :20], was[0][:, :, :, :20])  # position 20's block has got more rows
    cache.free([1, 4])
    cache.compact()
    for slot in (0, 2, 3):
        assert torch.equal(values(cache, slot), now[slot])
    used = int((cache.refs > 0).sum())
    assert (cache.refs[:used] > 0).all()
    short = PagedCache(1, 2, 1, 1, 16, page_size=16, dtype=E4M3)
    short.reserve([5, 0])
    short.append(*(torch.randn(1, 2, 5, 1, 16, device=DEV) for _ in range(2)), count=torch.tensor([5, 0], dtype=torch.int32, device=DEV))
    before = values(short, 0)
    assert short.fork([0], [1]).item() == 1 and torch.equal(values(short, 0), before)


def test_a_step_replays_from_a_graph():
    blocks, rotary, V, B = blocks_of(1), Rotary(64, 32, interleaved=True), 64, 2
    g = torch.Generator(device=DEV).manual_seed(6)
    embedding = torch.randn(V, 256, generator=g, device=DEV).to(BF)
    head = (torch.randn(256, V, generator=g, device=DEV) * 0.3).to(BF)
    settings = dict(temperature=torch.tensor([0.7, 1.0], device=DEV), top_p=torch.tensor([0.9, 1.0], device=DEV))

    def start():
        cache = PagedCache(1, B, 30, 4, 64, page_size=8, dtype=E4M3, block=8)
        for t in (cache.k, cache.v):
            t.view(torch.uint8).zero_()
        cache.reserve(torch.tensor([40, 60], dtype=torch.int32))
        extend(blocks, embedding[:20].expand(B, 20, 256).contiguous(), cache, rotary)
        return cache

    a, b = start(), start()
    us = torch.rand(5, B, generator=g, device=DEV)
    last, want = torch.tensor([1, 2], dtype=torch.int32, device=DEV), []
    for u in us:
        last, prob = step(blocks, embedding, head, a, last, u, rotary, **settings)
        want.append((last.clone(), prob.clone()))
    u, last = us[0].clone(), torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(blocks, embedding, head, start(), last, u, rotary, **settings)  # first calls outside the capture
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            token, prob = step(blocks, embedding, head, b, last, u, rotary, **settings)
            last.copy_(token)
    torch.cuda.current_stream().wait_stream(side)
    for i, w in enumerate(want):
        u.copy_(us[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(token, w[0]) and torch.equal(prob, w[1])
    assert torch.equal(a.lens, b.lens) and torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8))


def test_speculative_steps_on_an_8bit_cache():
    """Drafts that the model itself would take are accepted, and the cache goes on from them."""
    blocks, rotary, V, B = blocks_of(2), Rotary(64), 64, 2
    g = torch.Generator(device=DEV).manual_seed(9)
    embedding = torch.randn(V, 256, generator=g, device=DEV).to(BF)
    head = (torch.randn(256, V, generator=g, device=DEV) * 0.3).to(BF)
    cache = PagedCache(2, B, 40, 4, 64, page_size=16, dtype=E4M3)
    cache.reserve(100)
    extend(blocks, embedding[torch.randint(0, V, (B, 30), generator=g, device=DEV)], cache, rotary)
    last, accepted = torch.tensor([5, 6], dtype=torch.int32, device=DEV), 0
    for _ in range(4):
        drafts = torch.randint(0, V, (B, 3), generator=g, device=DEV).int()
        y, _, _ = decode(blocks, embedding[last.long()][:, None], cache, None, rotary)
        drafts[:, 0], _ = next_token(y[:, 0], head, torch.zeros(B, device=DEV), temperature=0.0)
        n = cache.lens.tolist()
        u = torch.rand(B, 4, generator=g, device=DEV)
        u[:, 0] = 0.0
        parents = torch.tensor([[-1, 0, -1]] * B, dtype=torch.int32, device=DEV)
        path, count, last = speculative_step(blocks, embedding, head, cache, last, drafts, u, parents, rotary=rotary)
        assert (count >= 1).all() and cache.lens.tolist() == [x + int(c) + 1 for x, c in zip(n, count)]
        accepted += int(count.sum())
    assert accepted >= 8


def test_refusals():
    with pytest.raises(ValueError):
        PagedCache(1, 2, 4, 4, 64, page_size=24, dtype=E4M3)  # blocks of 16
    with pytest.raises(ValueError):
        Rotary(64, 72)
    with pytest.raises(ValueError):
        Rotary(64, scaling="linear", factor=0.5)
