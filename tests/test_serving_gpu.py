"""nkilab.serving: decoding over the paged cache gives what the whole sequence gives at once."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nkilab import ops
from nkilab.model import BlockConfig, DecoderBlock, nki_forward
from nkilab.serving import PagedCache, decode, probabilities, speculative_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


def blocks_of(layers, dtype, d_model=256, heads=4, d_ff=384):
    torch.manual_seed(3)
    return [DecoderBlock(BlockConfig(d_model, heads, d_ff)).to(DEV).eval() for _ in range(layers)]


def whole(blocks, x):
    for b in blocks:
        x = nki_forward(b, x)
    return x


# fp32: two orders of the same sums through the layers; bf16: each layer rounds at the same
# places, but P and its sums differ in their last bit, which a layer's residual carries on
BOUND = {torch.float32: 2e-4, torch.bfloat16: 6e-2}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_chunks_of_a_prompt_equal_the_prompt(dtype):
    blocks = blocks_of(2, dtype)
    S, B = 150, 2
    x = torch.randn(B, S, 256, device=DEV).to(dtype)
    want = torch.stack([whole(blocks, x[b]) for b in range(B)])
    cache = PagedCache(2, B, 24, 4, 64, page_size=16, dtype=dtype)
    got, at = [], 0
    for n in (1, 64, 3, 81, 1):
        cache.reserve(n)
        y, k, v = decode(blocks, x[:, at:at + n], cache)
        cache.append(k, v)
        got.append(y)
        at += n
    assert at == S and cache.lens.tolist() == [S] * B and cache.missing.item() == 0
    err = (torch.cat(got, 1).float() - want.float()).abs().max() / want.float().abs().max()
    assert err < BOUND[dtype]


def test_a_path_of_a_tree_equals_its_sequence():
    """Every node of a tree gives what the sequence from the root to it gives."""
    blocks = blocks_of(1, torch.float32)
    prompt, tree = torch.randn(1, 20, 256, device=DEV), torch.randn(1, 7, 256, device=DEV)
    parents = [-1, 0, 0, 1, -1, 4, 3]
    cache = PagedCache(1, 1, 4, 4, 64, page_size=8, dtype=torch.float32)
    cache.reserve(20)
    cache.append(*decode(blocks, prompt, cache)[1:])
    y, k, v = decode(blocks, tree, cache, torch.tensor([parents], dtype=torch.int32, device=DEV))
    for i in range(7):
        chain, j = [], i
        while j >= 0:
            chain.insert(0, j)
            j = parents[j]
        want = whole(blocks, torch.cat([prompt[0], tree[0, chain]]))[-1]
        assert (y[0, i] - want).abs().max() / want.abs().max() < BOUND[torch.float32]


@pytest.mark.parametrize("tree", [False, True])
def test_speculative_steps_keep_what_was_accepted(tree):
    """After several steps on forked and freed slots, the cache holds the accepted tokens: one
    more pass over it equals the whole sequence at once."""
    dtype, V, B = torch.bfloat16, 64, 3
    blocks = blocks_of(2, dtype)
    g = torch.Generator(device=DEV).manual_seed(5)
    embedding = torch.randn(V, 256, generator=g, device=DEV).to(dtype)
    head = (torch.randn(256, V, generator=g, device=DEV) * 0.3).to(dtype)
    cache = PagedCache(2, B, 40, 4, 64, page_size=8, max_len=120, dtype=dtype)
    prompt = torch.randint(0, V, (B, 21), generator=g, device=DEV)
    cache.reserve(20)
    cache.append(*decode(blocks, embedding[prompt[:, :20]], cache)[1:])
    cache.fork([0], [2])
    prompt[2] = prompt[0]
    history = [prompt[b].tolist() for b in range(B)]
    last = prompt[:, 20].int()
    parents = torch.tensor([[-1, 0, -1, 2, 2, -2]] * B, dtype=torch.int32, device=DEV) if tree else None
    accepted = 0
    for step in range(6):
        cache.reserve(7)
        assert cache.missing.item() == 0
        drafts = torch.randint(0, V, (B, 6), generator=g, device=DEV).int()
        if step % 2:  # what the model likes best, so that some are accepted
            y, _, _ = decode(blocks, embedding[last.long()][:, None], cache)
            drafts[:, 0] = probabilities(y, head)[:, 0].argmax(-1).int()
        u = torch.rand(B, 7, generator=g, device=DEV)
        u[:, 0] *= 0.01
        path, count, last = speculative_step(blocks, embedding, head, cache, last, drafts, u, parents)
        for b in range(B):
            history[b] += [int(drafts[b, i]) for i in path[b].tolist() if i >= 0] + [int(last[b])]
        accepted += int(count.sum())
        if step == 3:
            cache.free([1])
            cache.compact()
            cache.fork([2], [1])
            history[1] = list(history[2])
            last[1] = last[2]
    assert accepted > 0
    assert cache.lens.tolist() == [len(h) - 1 for h in history]
    y, _, _ = decode(blocks, embedding[last.long()][:, None], cache)
    for b in range(B):
        want = whole(blocks, embedding[torch.tensor(history[b], device=DEV)])[-1].float()
        assert (y[b, 0].float() - want).abs().max() / want.abs().max() < BOUND[dtype]


def test_a_draft_without_an_earlier_parent_follows_the_last_token():
    """A parent that is the token itself or a later one counts as none, in every part of a step."""
    blocks = blocks_of(2, torch.float32)
    embedding, head = torch.randn(64, 256, device=DEV), torch.randn(256, 64, device=DEV) * 0.05
    prompt = torch.randn(1, 9, 256, device=DEV)
    drafts = torch.tensor([[3, 14, 15, 9, 26]], dtype=torch.int32, device=DEV)
    last = torch.tensor([5], dtype=torch.int32, device=DEV)
    uniforms = torch.tensor([[0.0] * 5 + [0.5]], device=DEV)  # a first child is always accepted
    got = []
    for parents in ([-1, 0, 1, -1, 3], [0, 0, 1, 4, 3]):
        cache = PagedCache(2, 1, 4, 4, 64, page_size=8, dtype=torch.float32)
        cache.reserve(20)
        cache.append(*decode(blocks, prompt, cache)[1:])
        tree = torch.tensor([parents], dtype=torch.int32, device=DEV)
        out = speculative_step(blocks, embedding, head, cache, last, drafts, uniforms, tree)
        pages = cache.k[:, cache.tables[0, :3].long()]  # [layers, 3, heads, page, head_dim]
        got.append([*out, cache.lens, pages.transpose(2, 3).flatten(1, 2)[:, :int(cache.lens)]])
    assert got[0][0].tolist() == [[0, 1, 2, -1, -1]]
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_a_step_replays_from_a_graph():
    dtype, V, B = torch.bfloat16, 64, 2
    blocks = blocks_of(1, dtype)
    g = torch.Generator(device=DEV).manual_seed(6)
    embedding = torch.randn(V, 256, generator=g, device=DEV).to(dtype)
    head = (torch.randn(256, V, generator=g, device=DEV) * 0.3).to(dtype)

    def start():
        cache = PagedCache(1, B, 30, 4, 64, page_size=8, dtype=dtype)
        cache.reserve(torch.tensor([30, 50], dtype=torch.int32))
        cache.append(*decode(blocks, embedding[:20].expand(B, 20, 256).contiguous(), cache)[1:])
        return cache

    drafts = torch.randint(0, V, (B, 3), generator=g, device=DEV).int()
    last, u = torch.tensor([1, 2], dtype=torch.int32, device=DEV), torch.rand(B, 4, generator=g, device=DEV)
    a, b = start(), start()
    want = []
    for _ in range(3):
        want.append([t.clone() for t in speculative_step(blocks, embedding, head, a, last, drafts, u)])
        a.reserve(4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        c = start()
        speculative_step(blocks, embedding, head, c, last, drafts, u)  # first calls outside the capture
        c.reserve(torch.full_like(c.lens, 4))
        side.synchronize()
        extra = torch.full_like(b.lens, 4)
        with torch.cuda.graph(graph, stream=side):
            got = speculative_step(blocks, embedding, head, b, last, drafts, u)
            b.reserve(extra)
    for w in want:
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, w):
            assert torch.equal(x, y)
    assert torch.equal(a.lens, b.lens) and torch.equal(a.tables, b.tables)


def test_a_length_ends_with_the_pages():
    """After a reserve that failed, rows without a page are dropped and not counted: no later
    attention reads positions that were never written."""
    blocks = blocks_of(1, torch.float32)
    x = torch.randn(2, 20, 256, device=DEV)
    cache = PagedCache(1, 2, 4, 4, 64, page_size=8, dtype=torch.float32)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    cache.reserve([8, 16])
    assert cache.reserve(20).item() > 0
    _, k, v = decode(blocks, x, cache)
    cache.append(k, v)
    assert cache.lens.tolist() == [8, 16]
    path = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    cache.append(k[:, :, :3], v[:, :, :3], path, torch.tensor([3, 2], dtype=torch.int32, device=DEV))
    assert cache.lens.tolist() == [8, 16]
    assert cache.reserve([1, 0]).item() == 0  # the last free page, with whatever it holds
    y, _, _ = decode(blocks, x[:, :1], cache)
    for b, n in enumerate((8, 16)):
        want = whole(blocks, torch.cat([x[b, :n], x[b, :1]]))[-1]
        assert (y[b, 0] - want).abs().max() / want.abs().max() < BOUND[torch.float32]


def test_refusals():
    with pytest.raises(ValueError):
        PagedCache(1, 0, 4, 4, 64)
    cache = PagedCache(1, 2, 4, 4, 64, page_size=8)
    assert cache.reserve(17).item() == 2  # 3 pages for each of two slots, 4 there are
    assert cache.refs.sum().item() == 0
