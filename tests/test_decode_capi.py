"""Argument checks of the decoding entry points of the C ABI (CPU only: no call here reaches a
kernel launch)."""
from __future__ import annotations

import ctypes

import pytest

FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below fails validation first
ODD = ctypes.c_void_p(4104)   # 8-byte but not 16-byte aligned


@pytest.fixture(scope="module")
def N():
    from nkilab import _native

    return _native


def strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def tree(N, **kw):
    a = dict(q=FAKE, qs=None, k=FAKE, v=FAKE, ns=None, kc=FAKE, vc=FAKE, cs=None, tables=FAKE, lens=FAKE, parents=None,
             out=FAKE, ws=None, wsb=0, B=2, T=4, H=8, Hkv=2, d=64, P=10, page=16, M=4, scale=0.1, dt=N.BFLOAT16)
    assert not set(kw) - set(a)
    a.update(kw)
    return N.lib.nkl_attention_tree(*a.values(), None)


def test_attention_tree_refusals(N):
    assert tree(N, dt=5) == N.ERR_DTYPE
    assert tree(N, T=129) == N.ERR_SHAPE and b"129" in N.lib.nkl_last_error()
    assert tree(N, Hkv=3) == N.ERR_SHAPE
    assert tree(N, Hkv=0) == N.ERR_SHAPE
    assert tree(N, d=68) == N.ERR_SHAPE
    assert tree(N, d=136) == N.ERR_SHAPE
    assert tree(N, page=0) == N.ERR_SHAPE
    assert tree(N, M=0) == N.ERR_SHAPE
    assert tree(N, P=0) == N.ERR_SHAPE
    assert tree(N, B=-1) == N.ERR_SHAPE
    assert tree(N, page=65536, M=1 << 20) == N.ERR_SHAPE
    for name in ("q", "k", "v", "kc", "vc", "tables", "lens", "out"):
        assert tree(N, **{name: None}) == N.ERR_ARG
    for name in ("q", "k", "v", "kc", "vc", "out"):
        assert tree(N, **{name: ODD}) == N.ERR_ALIGN
    assert tree(N, qs=strides(512, 130, 64)) == N.ERR_ALIGN
    assert tree(N, cs=strides(-2048, 1024, 64)) == N.ERR_ALIGN
    need = N.lib.nkl_attention_tree_workspace_size(2, 4, 8, 2, 64, 16, 4000, N.FLOAT32)
    assert need > 0  # else the calls below would launch
    assert tree(N, M=4000, dt=N.FLOAT32) == N.ERR_ARG and b"workspace" in N.lib.nkl_last_error()
    assert tree(N, M=4000, dt=N.FLOAT32, ws=FAKE, wsb=need - 1) == N.ERR_ARG
    assert tree(N, M=4000, dt=N.FLOAT32, ws=ctypes.c_void_p(4096 + 16), wsb=need) == N.ERR_ALIGN


def test_attention_tree_nothing_to_do(N):
    assert tree(N, B=0, q=None) == N.OK
    assert tree(N, T=0, q=None) == N.OK
    assert N.lib.nkl_attention_tree_workspace_size(0, 4, 8, 2, 64, 16, 4, N.BFLOAT16) == 0
    assert N.lib.nkl_attention_tree_workspace_size(2, 4, 8, 3, 64, 16, 4, N.BFLOAT16) == 0
    assert N.lib.nkl_attention_tree_workspace_size(2, 4, 8, 2, 64, 16, 400, N.FLOAT32) > 0


def append(N, **kw):
    a = dict(k=FAKE, v=FAKE, ks=None, kc=FAKE, vc=FAKE, cs=None, tables=FAKE, lens=FAKE, path=None, count=None,
             out=FAKE, L=1, B=2, T=3, Hkv=2, d=64, P=10, page=16, M=4, dt=N.BFLOAT16)
    assert not set(kw) - set(a)
    a.update(kw)
    return N.lib.nkl_cache_append(*a.values(), None)


def test_append_refusals(N):
    assert append(N, dt=9) == N.ERR_DTYPE
    assert append(N, d=60) == N.ERR_SHAPE
    for name in ("L", "Hkv", "P", "page", "M"):
        assert append(N, **{name: 0}) == N.ERR_SHAPE
    assert append(N, B=-1) == N.ERR_SHAPE
    assert append(N, T=-1) == N.ERR_SHAPE
    for name in ("k", "v", "kc", "vc", "tables", "lens", "out"):
        assert append(N, **{name: None}) == N.ERR_ARG
    for name in ("k", "v", "kc", "vc"):
        assert append(N, **{name: ODD}) == N.ERR_ALIGN
    assert append(N, ks=strides(1000, 384, 129, 64)) == N.ERR_ALIGN
    assert append(N, cs=strides(20480, 2048, 1024, 32)) == N.ERR_ALIGN
    assert append(N, B=0) == N.OK


def test_page_operation_refusals(N):
    L = N.lib
    assert L.nkl_cache_reserve(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 0, 2, 10, 16, 4, None) == N.ERR_ARG
    assert L.nkl_cache_reserve(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 999, 2, 10, 0, 4, None) == N.ERR_SHAPE
    assert L.nkl_cache_reserve(None, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 999, 2, 10, 16, 4, None) == N.ERR_ARG
    n = L.nkl_cache_fork_workspace_size(4, 3)
    assert n >= (4 + 2 * 3) * 4 and n % 256 == 0

    def fork(**kw):
        a = dict(kc=FAKE, vc=FAKE, cs=None, tables=FAKE, lens=FAKE, refs=FAKE, src=FAKE, dst=FAKE, to=FAKE, lo=FAKE,
                 ro=FAKE, missing=FAKE, ws=FAKE, wsb=n, F=3, L=1, B=4, Hkv=2, d=64, P=10, page=16, M=4, dt=N.BFLOAT16)
        a.update(kw)
        return L.nkl_cache_fork(*a.values(), None)

    assert fork(wsb=n - 1) == N.ERR_ARG
    assert fork(ws=None) == N.ERR_ARG
    assert fork(src=None) == N.ERR_ARG
    assert fork(F=-1) == N.ERR_SHAPE
    assert fork(B=0) == N.ERR_SHAPE
    assert fork(dt=7) == N.ERR_DTYPE
    assert fork(vc=ODD) == N.ERR_ALIGN
    assert L.nkl_cache_free(FAKE, FAKE, FAKE, None, FAKE, FAKE, FAKE, 2, 4, 10, 4, None) == N.ERR_ARG
    assert L.nkl_cache_free(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 4, 0, 4, None) == N.ERR_SHAPE
    m = L.nkl_cache_compact_workspace_size(10)
    assert m >= 31 * 4
    assert L.nkl_cache_compact(FAKE, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, m - 1, 1, 4, 2, 64, 10, 16, 4, N.BFLOAT16,
                               None) == N.ERR_ARG
    assert L.nkl_cache_compact(FAKE, FAKE, None, FAKE, None, FAKE, FAKE, FAKE, m, 1, 4, 2, 64, 10, 16, 4, N.BFLOAT16,
                               None) == N.ERR_ARG


def test_verify_refusals(N):
    def verify(**kw):
        a = dict(p=FAKE, q=None, tokens=FAKE, u=FAKE, parents=None, path=FAKE, count=FAKE, token=FAKE, B=2, T=3, V=100,
                 dt=N.FLOAT32)
        a.update(kw)
        return N.lib.nkl_verify_drafts(*a.values(), None)

    assert verify(dt=3) == N.ERR_DTYPE
    assert verify(V=0) == N.ERR_SHAPE
    assert verify(T=129) == N.ERR_SHAPE
    assert verify(T=-1) == N.ERR_SHAPE
    assert verify(B=-1) == N.ERR_SHAPE
    assert verify(q=FAKE, parents=FAKE) == N.ERR_ARG
    for name in ("p", "tokens", "u", "path", "count", "token"):
        assert verify(**{name: None}) == N.ERR_ARG
    assert verify(p=ctypes.c_void_p(4097)) == N.ERR_ALIGN
    assert verify(B=0, p=None) == N.OK


def test_wrappers_take_no_cpu_tensors():
    import torch

    from nkilab import ops

    i = torch.zeros(1, 1, dtype=torch.int32)
    x = torch.zeros(1, 1, 2, 64)
    with pytest.raises(NotImplementedError):
        ops.attention_tree(x, x, x, x, x, i, i[0])
    with pytest.raises(NotImplementedError):
        ops.verify_drafts(torch.ones(1, 2, 4), i, torch.zeros(1, 2))
    with pytest.raises(NotImplementedError):
        ops.cache_free(i, i[0], i[0], i[0])


def test_shapes_without_a_gpu():
    """The operators' shape functions: what a trace or an allocation ahead of the call sees."""
    import torch

    from nkilab import ops

    def m(*shape, dtype=torch.int32):
        return torch.empty(shape, dtype=dtype, device="meta")

    bf = torch.bfloat16
    L, B, T, H, Hkv, d, P, page, M, V = 3, 2, 5, 8, 2, 64, 20, 16, 7, 50
    cache = m(L, P, Hkv, page, d, dtype=bf)
    tables, lens, refs = m(B, M), m(B), m(P)
    out = ops.attention_tree(m(B, T, H, d, dtype=bf), m(B, T, Hkv, d, dtype=bf), m(B, T, Hkv, d, dtype=bf), cache[0], cache[0],
                             tables, lens, m(B, T))
    assert out.shape == (B, T, H, d) and out.dtype == bf
    rows = m(L, B, T, Hkv, d, dtype=bf)
    assert ops.cache_append(rows, rows, cache, cache, tables, lens).shape == (B,)
    assert [t.shape for t in ops.cache_reserve(tables, lens, refs, m(B), page)] == [(B, M), (P,), (1,)]
    assert [t.shape for t in ops.cache_fork(cache, cache, tables, lens, refs, m(1), m(1))] == [(B, M), (B,), (P,), (1,)]
    assert [t.shape for t in ops.cache_free(tables, lens, refs, m(1))] == [(B, M), (B,), (P,)]
    assert [t.shape for t in ops.cache_compact(cache, cache, tables, refs)] == [(B, M), (P,)]
    got = ops.verify_drafts(m(B, T + 1, V, dtype=torch.float32), m(B, T), m(B, T + 1, dtype=torch.float32))
    assert [t.shape for t in got] == [(B, T), (B,), (B,)] and all(t.dtype == torch.int32 for t in got)


def test_a_backward_pass_raises():
    """The attention is for decoding: a gradient through it is refused, never left out."""
    import torch

    from nkilab import ops

    def m(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="meta")

    i = torch.int32
    args = [m(1, 2, 4, 64), m(1, 2, 2, 64), m(1, 2, 2, 64), m(9, 2, 16, 64), m(9, 2, 16, 64)]
    assert not ops.attention_tree(*args, m(1, 3, dtype=i), m(1, dtype=i)).requires_grad
    for x in args:
        x.requires_grad_()
        out = ops.attention_tree(*args, m(1, 3, dtype=i), m(1, dtype=i))
        assert out.requires_grad
        with pytest.raises(RuntimeError, match="attention_tree"):
            out.sum().backward()
        with torch.no_grad():
            assert not ops.attention_tree(*args, m(1, 3, dtype=i), m(1, dtype=i)).requires_grad
        x.requires_grad_(False)
