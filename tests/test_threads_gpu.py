"""Host threads that queue on one stream: each call's launches stay together, and no call reads what
another one left in a workspace."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from nkilab import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def i32(x):
    return torch.from_numpy(np.ascontiguousarray(x)).int().to(DEV)


def tree(seed, dtype, T, lens, page=16, H=8, Hkv=2, d=64):
    """Long rows over few heads: their key ranges are cut, and a second launch joins the pieces."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = np.random.RandomState(seed)
    need = [-(-n // page) for n in lens]
    order = r.permutation(sum(need))
    tables = np.full((len(lens), max(need)), -1)
    for b, n in enumerate(need):
        tables[b, :n] = order[sum(need[:b]):][:n]
    kc, vc = (torch.randn(sum(need), Hkv, page, d, generator=g, device=DEV).to(dtype) for _ in range(2))
    q, k, v = (torch.randn(len(lens), T, h, d, generator=g, device=DEV).to(dtype) for h in (H, Hkv, Hkv))
    tables, lens = i32(tables), i32(lens)
    return lambda: (ops.attention_tree(q, k, v, kc, vc, tables, lens),)


def fork(seed, B, P):
    r = np.random.RandomState(seed)
    tables, refs = np.full((B, 3), -1), np.zeros(P, int)
    pages = r.permutation(P)[:6]
    lens = np.zeros(B, int)
    lens[:3] = 11, 16, 5
    tables[0, :2], tables[1, :2], tables[2, 0] = pages[:2], pages[2:4], pages[4]
    refs[pages[:5]] = 1
    kc = torch.randn(1, P, 1, 8, 8, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)
    tables, lens, refs = i32(tables), i32(lens), i32(refs)
    src, dst = i32(r.randint(0, 3, B - 3)), i32(r.permutation(np.arange(3, B)))

    def call():
        k, v = kc.clone(), kc + 1
        return *ops.cache_fork(k, v, tables, lens, refs, src, dst), k, v

    return call


def compact(seed, P):
    r = np.random.RandomState(seed)
    refs = (r.rand(P) < 0.4) * r.randint(1, 4, P)
    kc = torch.arange(P, device=DEV, dtype=torch.float32).view(1, P, 1, 1, 1).expand(2, P, 1, 1, 4).contiguous()
    tables, refs = i32(np.where(refs > 0, np.arange(P), -1).reshape(1, P)), i32(refs)

    def call():
        k, v = kc.clone(), kc + 0.5
        return *ops.cache_compact(k, v, tables, refs), k, v

    return call


def prompt(seed, H, S, strided=False):
    """Long prompts of few heads, whose key ranges are split over the SMs."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    q, k, v = (torch.randn(H, S, 64, generator=g, device=DEV).to(BF) for _ in range(3))

    def call():
        if not strided:
            return (ops.attention(q, k, v),)
        out = torch.empty_like(q)
        torch.ops.nkilab.attention_strided_(q, k, v, out, 0.125)
        return (out,)

    return call


PAIRS = {
    "attention": lambda: (prompt(11, 2, 2048), prompt(12, 3, 1408)),
    "attention strided": lambda: (prompt(13, 2, 2048, True), prompt(14, 1, 4096)),
    "attention_tree bf16": lambda: (tree(1, BF, 1, [5000, 4000]), tree(2, BF, 40, [900, 3000, 77, 2500])),
    "attention_tree f32": lambda: (tree(3, torch.float32, 1, [3000]), tree(4, torch.float32, 5, [700, 2000, 1500])),
    "cache_fork": lambda: (fork(5, 900, 5000), fork(6, 2500, 6000)),
    "cache_compact": lambda: (compact(7, 9001), compact(8, 12000)),
    "mixed": lambda: (tree(9, BF, 3, [6000]), compact(10, 9500)),
}


@pytest.mark.parametrize("name", list(PAIRS))
def test_two_threads_on_one_stream(name):
    calls = PAIRS[name]()
    want = [c() for c in calls]
    torch.cuda.synchronize()
    n, start, got = 200, threading.Barrier(2), [[], []]

    def work(i):
        start.wait(60)
        for _ in range(n):
            got[i].append([x.equal(y) for x, y in zip(calls[i](), want[i])] if len(got[i]) % 50 == 49 else calls[i]())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == n
        for out in got[i]:
            assert all(x if isinstance(x, bool) else torch.equal(x, y) for x, y in zip(out, want[i]))
