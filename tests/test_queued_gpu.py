"""Kernels queued behind the one that writes their input: each may begin before that one ends, and
has to read what it wrote, not what the memory held before."""
from __future__ import annotations

import pytest
import torch

from nkilab import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
M, K, N = 4096, 512, 2048


def readers():
    """Nothing of theirs runs between the product and the kernel that reads it."""
    ones = torch.ones(N, device=DEV, dtype=BF)
    cache = torch.zeros(2, 1, M // 64, N // 128, 64, 128, device=DEV, dtype=BF)
    tables, lens = torch.arange(M // 64, device=DEV).int()[None], torch.zeros(1, dtype=torch.int32, device=DEV)

    def append(x):
        k = x.view(1, 1, M, N // 128, 128)
        ops.cache_append(k, k, cache[0], cache[1], tables, lens)
        return cache.clone()

    return {
        "rmsnorm": lambda x: ops.rmsnorm(x, ones),
        "softmax": ops.softmax,
        "swiglu": lambda x: ops.swiglu(x, x),
        "add_rmsnorm": lambda x: torch.cat(torch.ops.nkilab.add_rmsnorm(x, x, ones, 1e-6)),
        "rope": lambda x: ops.rope(x.view(16, -1, 128)),
        "cache_append": append,
    }


NAMES = ["rmsnorm", "softmax", "swiglu", "add_rmsnorm", "rope", "cache_append"]


@pytest.mark.parametrize("name", NAMES)
def test_reads_what_the_kernel_before_wrote(name):
    read = readers()[name]
    g = torch.Generator().manual_seed(1)
    a = (torch.rand(M, K, generator=g) * 2 - 1).to(DEV, BF)
    b = (torch.rand(K, N, generator=g) * 2 - 1).to(DEV, BF)
    x = ops.matmul(a, b)
    torch.cuda.synchronize()
    want = read(x)
    torch.cuda.synchronize()
    del x
    busy = torch.randn(4096, 4096, device=DEV, dtype=BF)
    got = []
    for i in range(12):
        if i % 6 == 0:  # so that the host is ahead of the GPU
            for _ in range(8):
                busy @ busy
        old = torch.full((M, N), 7.0, device=DEV, dtype=BF)
        del old  # the product takes its place
        got.append(read(ops.matmul(a, b)))
    torch.cuda.synchronize()
    for y in got:
        assert torch.equal(y, want)


@pytest.mark.parametrize("name", ["matmul", "attention", "attention_tree"])
def test_tiles_of_what_the_kernel_before_wrote(name):
    """The same where the reader fetches tiles, the first of them asked for before it may read."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(16, 1024, 128, generator=g).to(DEV, BF)
    w = (torch.randn(2048, 1024, generator=g) * 0.02).to(DEV, BF)
    ones = torch.ones(2048, device=DEV, dtype=BF)
    kc = torch.randn(16, 16, 64, 128, generator=g).to(DEV, BF)
    tables, lens = torch.arange(16, device=DEV).int()[None], torch.tensor([1000], device=DEV).int()

    def write():
        return ops.rmsnorm(x.view(-1, 2048), ones) if name == "matmul" else ops.rope(x)

    def read(h):
        if name == "matmul":
            return ops.matmul(h, w)
        if name == "attention":
            return ops.attention(h, h, h)
        q = h.view(16, 16, 64, 128)[None, :, :, 0].transpose(1, 2)  # 16 tokens of 16 heads
        return ops.attention_tree(q, q, q, kc, kc, tables, lens)

    h = write()
    torch.cuda.synchronize()
    want = read(h)
    torch.cuda.synchronize()
    del h
    busy = torch.randn(4096, 4096, device=DEV, dtype=BF)
    got = []
    for i in range(12):
        if i % 6 == 0:
            for _ in range(8):
                busy @ busy
        old = torch.full((x.numel(),), 7.0, device=DEV, dtype=BF)
        del old
        got.append(read(write()))
    torch.cuda.synchronize()
    for y in got:
        assert torch.equal(y, want)
