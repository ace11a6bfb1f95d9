"""Rotary positions and the 8-bit cache where their kernels change hands: the most rows that one takes, tiles and
pieces that end on a border, blocks of a few positions, groups of tokens wider than a pass, calls of two threads."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from nkilab import ops
from test_attention_8bit_gpu import BF, DEV, E4M3, F32, check, exact, i32, run, setup
from test_decode_gpu import random_trees
from test_rotary_gpu import check as check_rotary
from test_rotary_gpu import freqs_of, turned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[0], [1, 127, 128, 129], [9000, 0, 640, 641, 511], [127] * 40])
@pytest.mark.parametrize("T,H,Hkv,d,page,block", [(16, 3, 3, 128, 64, 4), (2, 32, 4, 128, 8, 2), (1, 16, 1, 64, 24, 3), (8, 4, 4, 128, 16, 1),
                                                  (3, 10, 2, 64, 128, 128), (1, 8, 1, 128, 256, 16)])
def test_rows_that_share_a_tile(T, H, Hkv, d, page, block, lens):
    """Up to 16 query rows to a key/value head: lengths around tiles, drafted tokens alone, blocks that split fours."""
    x = setup(len(lens), T, H, Hkv, d, page, block, lens, BF, seed=T + len(lens))
    for parents in (None, i32(random_trees(np.random.RandomState(T), len(lens), T).tolist())):
        check(run(x, parents), *exact(x, parents), BF)


@pytest.mark.parametrize("T,d,page,dtype", [(1, 128, 64, BF), (4, 64, 32, BF), (40, 128, 64, BF), (2, 96, 16, BF), (2, 128, 64, F32)])
def test_a_block_that_grows_changes_no_result(T, d, page, dtype):
    """A row behind a sequence's last one makes its block grow by 2^3. The values are small whole numbers and so stay what
    they are, and all weights are over 2^-12 of the largest, so that f16 holds them to the same place."""
    g = torch.Generator(device=DEV).manual_seed(4)
    B, H, Hkv, n = 2, 8, 4, 300
    M = n // page + 2
    kc, vc = (torch.zeros(B * M, Hkv, page, d, dtype=E4M3, device=DEV) for _ in range(2))
    ks, vs = (torch.full((B * M, Hkv, page // 8), 127, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu) for _ in range(2))
    tables, lens = torch.arange(B * M, device=DEV).view(B, M).int(), i32([n, n - 37])
    rows = [torch.randint(-7, 8, (1, B, n, Hkv, d), generator=g, device=DEV).to(dtype) for _ in range(2)]
    ops.cache_append(*rows, kc[None], vc[None], tables, i32([0, 0]), None, lens, ks[None], vs[None])
    q, k, v = torch.randn(B, T, H + 2 * Hkv, d, generator=g, device=DEV).to(dtype).split([H, Hkv, Hkv], 2)
    x = (q * 0.05, k * 0.05, v, kc, vc, tables, lens, ks, vs)
    want, before = run(x), ks.view(torch.uint8).clone()
    more = [torch.full((1, B, 1, Hkv, d), 56.0, device=DEV, dtype=dtype) for _ in range(2)]
    ops.cache_append(*more, kc[None], vc[None], tables, lens, None, None, ks[None], vs[None])
    assert not torch.equal(ks.view(torch.uint8), before)
    assert torch.equal(run(x), want)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,d,part,dtype", [(2, 5003, 3, 256, 256, F32), (2, 5003, 3, 256, 16, F32), (3, 3301, 5, 256, 256, BF), (3, 3301, 2, 96, 24, BF)])
def test_rotary_of_many_tokens(B, T, H, d, part, dtype, interleaved):
    """Groups of eight tokens, of which a pass over the threads takes fewer, or that end in a shorter one."""
    x = torch.randn(B, T, H, d, device=DEV).to(dtype)
    start, f = torch.randint(0, 1 << 20, (B,), device=DEV).int(), freqs_of(part)
    check_rotary(ops.rotary(x, start, f, interleaved=interleaved), *turned(x, start[:, None] + torch.arange(T, device=DEV), f, interleaved), dtype)


def test_two_threads_on_one_stream_and_on_two():
    """Pieces of cut sequences meet in a workspace that calls at a time must not share."""
    cases = [setup(2, T, 32, 8, 128, 64, 16, [30000, 20], BF, seed=T) for T in (1, 4, 20)]
    want = [run(x) for x in cases]
    torch.cuda.synchronize()
    for streams in ([torch.cuda.current_stream()] * 3, [torch.cuda.Stream() for _ in range(3)]):
        bad = []

        def work(x, y, stream):
            with torch.cuda.stream(stream):
                for _ in range(30):
                    if not torch.equal(run(x), y):
                        bad.append(1)

        threads = [threading.Thread(target=work, args=(*c, s)) for c, s in zip(zip(cases, want), streams)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not bad


def test_captured_with_its_gradient():
    """Rotary there and back in one graph, replayed with other inputs."""
    x = torch.randn(2, 70, 6, 64, device=DEV)
    g, f, at = torch.randn_like(x), freqs_of(64), i32([5, 900])

    def both():
        y = x.detach().requires_grad_()
        out = ops.rotary(y, at, f)
        return out.detach(), torch.autograd.grad(out, y, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, back = both()
    x.normal_()
    at.add_(77)
    graph.replay()
    want = both()
    assert torch.equal(y, want[0]) and torch.equal(back, want[1])
