"""Argument checks of the operators around a decoding step, their shape functions and their host
arithmetic (CPU only: no call here reaches a kernel launch)."""
from __future__ import annotations

import ctypes
import math

import pytest

FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below fails validation first
ODD = ctypes.c_void_p(4104)   # 8-byte but not 16-byte aligned


@pytest.fixture(scope="module")
def N():
    from nkilab import _native

    return _native


def strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def rotary(N, **kw):
    a = dict(x=FAKE, xs=None, positions=FAKE, parents=None, freqs=FAKE, out=FAKE, B=2, T=3, H=4, d=64, r=32, per=0, inter=0,
             inv=0, mag=1.0, dt=N.BFLOAT16)
    assert not set(kw) - set(a)
    a.update(kw)
    return N.lib.nkl_rotary(*a.values(), None)


def test_rotary_refusals(N):
    assert rotary(N, dt=4) == N.ERR_DTYPE
    for kw in (dict(d=60), dict(d=264), dict(r=0), dict(r=12), dict(r=72), dict(H=0), dict(B=-1), dict(T=-1)):
        assert rotary(N, **kw) == N.ERR_SHAPE
    for name in ("x", "positions", "freqs", "out"):
        assert rotary(N, **{name: None}) == N.ERR_ARG
    assert rotary(N, parents=FAKE, per=1) == N.ERR_ARG
    assert rotary(N, parents=FAKE, T=129) == N.ERR_ARG and b"128" in N.lib.nkl_last_error()
    for name in ("x", "out"):
        assert rotary(N, **{name: ODD}) == N.ERR_ALIGN
    assert rotary(N, xs=strides(768, 260, 64)) == N.ERR_ALIGN
    assert rotary(N, xs=strides(768, 256, -64)) == N.ERR_ALIGN
    assert rotary(N, B=0, x=None) == N.OK
    assert rotary(N, T=0, x=None) == N.OK


def append(N, **kw):
    a = dict(q=FAKE, qs=None, k=FAKE, v=FAKE, ns=None, kc=FAKE, vc=FAKE, cs=None, ks=FAKE, vs=FAKE, tables=FAKE, lens=FAKE,
             count=None, freqs=FAKE, qo=FAKE, ko=FAKE, B=2, T=3, H=8, Hkv=2, d=64, r=64, P=10, page=16, M=4, block=16, inter=0,
             mag=1.0, dt=N.BFLOAT16)
    assert not set(kw) - set(a)
    a.update(kw)
    return N.lib.nkl_rotary_append(*a.values(), None)


def test_rotary_append_refusals(N):
    assert append(N, dt=4) == N.ERR_DTYPE
    for kw in (dict(d=72), dict(d=144, r=144), dict(r=0), dict(r=72), dict(block=0), dict(block=5), dict(block=32), dict(page=0),
               dict(M=0), dict(P=0), dict(Hkv=0), dict(H=0), dict(page=65536, M=1 << 20)):
        assert append(N, **kw) == N.ERR_SHAPE
    for name in ("q", "k", "v", "kc", "vc", "tables", "lens", "freqs", "qo", "ko", "ks", "vs"):
        assert append(N, **{name: None}) == N.ERR_ARG
    for name in ("q", "k", "v", "kc", "vc", "qo", "ko"):
        assert append(N, **{name: ODD}) == N.ERR_ALIGN
    assert append(N, cs=strides(2048, 1024, 72)) == N.ERR_ALIGN
    assert append(N, ns=strides(384, 128, 63)) == N.ERR_ALIGN
    assert append(N, B=0, q=None) == N.OK
    assert append(N, T=0, q=None) == N.OK


def test_append_8bit_refusals(N):
    def call(**kw):
        a = dict(k=FAKE, v=FAKE, ns=None, kc=FAKE, vc=FAKE, cs=None, ks=FAKE, vs=FAKE, tables=FAKE, lens=FAKE, path=None,
                 count=None, out=FAKE, L=2, B=2, T=3, Hkv=2, d=64, P=10, page=16, M=4, block=8, dt=N.BFLOAT16)
        assert not set(kw) - set(a)
        a.update(kw)
        return N.lib.nkl_cache_append_8bit(*a.values(), None)

    assert call(dt=9) == N.ERR_DTYPE
    for kw in (dict(d=72), dict(d=256), dict(L=0), dict(Hkv=0), dict(P=0), dict(page=0), dict(M=0), dict(block=3), dict(B=-1), dict(T=-1)):
        assert call(**kw) == N.ERR_SHAPE
    for name in ("k", "v", "kc", "vc", "ks", "vs", "tables", "lens", "out"):
        assert call(**{name: None}) == N.ERR_ARG
    for name in ("k", "v", "kc", "vc"):
        assert call(**{name: ODD}) == N.ERR_ALIGN
    assert call(B=0) == N.OK


def test_shapes_without_a_gpu():
    import torch

    from nkilab import ops

    def m(*shape, dtype=torch.int32):
        return torch.empty(shape, dtype=dtype, device="meta")

    bf = torch.bfloat16
    B, T, H, Hkv, d = 2, 5, 8, 2, 64
    x, k = m(B, T, H, d, dtype=bf), m(B, T, Hkv, d, dtype=bf)
    assert ops.rotary(x, m(B), m(16, dtype=torch.float64)).shape == x.shape
    c, s = m(20, Hkv, 16, d, dtype=torch.float8_e4m3fn), m(20, Hkv, 2, dtype=torch.float8_e8m0fnu)
    q2, k2 = ops.rotary_append(x, k, k, c, c, m(B, 3), m(B), m(32, dtype=torch.float64), k_scales=s, v_scales=s)
    assert q2.shape == x.shape and k2.shape == k.shape and q2.dtype == bf
    assert ops.cache_append(k, k, c, c, m(B, 3), m(B), None, None, s, s).shape == (B,)
    with pytest.raises(ValueError):
        ops.cache_append(k, k, c, c, m(B, 3), m(B), None, None, s)


def test_rotary_frequencies():
    import torch

    from nkilab import ops

    f, m = ops.rotary_frequencies(64, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and m == 1.0
    assert f[0] == 1.0 and f[16].item() == pytest.approx(0.01, rel=1e-12)
    g, m = ops.rotary_frequencies(64, 10000.0, "linear", 4.0, device="cpu")
    assert torch.equal(g, f / 4) and m == 1.0
    g, m = ops.rotary_frequencies(64, 10000.0, "ntk", 8.0, device="cpu")
    assert g[0] == 1.0 and g[-1].item() == pytest.approx(f[-1].item() / 8, rel=1e-12)
    g, m = ops.rotary_frequencies(64, 10000.0, "yarn", 8.0, 4096, device="cpu")
    assert m == pytest.approx(0.1 * math.log(8) + 1)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 8, rtol=1e-14)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (g[mid] < f[mid]).all() and (g[mid] > f[mid] / 8).all()
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="cubic"), dict(rotary_dim=8, factor=0.5),
                dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, scaling="yarn"), dict(rotary_dim=2, scaling="ntk")):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad, device="cpu")


def test_wrappers_take_no_cpu_tensors():
    import torch

    from nkilab import ops

    x, i = torch.zeros(1, 1, 2, 64), torch.zeros(1, dtype=torch.int32)
    f = torch.ones(32, dtype=torch.float64)
    with pytest.raises(NotImplementedError):
        ops.rotary(x, i, f)
    with pytest.raises(NotImplementedError):
        ops.rotary_append(x, x, x, x, x, i[None], i, f)


def test_attention_8bit_refusals(N):
    def call(**kw):
        a = dict(q=FAKE, qs=None, k=FAKE, v=FAKE, ns=None, kc=FAKE, vc=FAKE, cs=None, ks=FAKE, vs=FAKE, tables=FAKE, lens=FAKE,
                 parents=None, out=FAKE, ws=None, wsb=0, B=2, T=4, H=8, Hkv=2, d=64, P=10, page=16, M=4, block=8, scale=0.1,
                 dt=N.BFLOAT16)
        assert not set(kw) - set(a)
        a.update(kw)
        return N.lib.nkl_attention_tree_8bit(*a.values(), None)

    assert call(dt=5) == N.ERR_DTYPE
    for kw in (dict(T=129), dict(Hkv=3), dict(Hkv=0), dict(d=72), dict(d=144), dict(page=0), dict(M=0), dict(P=0), dict(B=-1),
               dict(block=0), dict(block=3), dict(block=32), dict(page=65536, M=1 << 20)):
        assert call(**kw) == N.ERR_SHAPE
    for name in ("q", "k", "v", "kc", "vc", "ks", "vs", "tables", "lens", "out"):
        assert call(**{name: None}) == N.ERR_ARG
    for name in ("q", "k", "v", "kc", "vc", "out"):
        assert call(**{name: ODD}) == N.ERR_ALIGN
    assert call(qs=strides(512, 130, 64)) == N.ERR_ALIGN
    assert call(cs=strides(2048, 1024, 72)) == N.ERR_ALIGN
    need = N.lib.nkl_attention_tree_8bit_workspace_size(2, 4, 8, 2, 64, 16, 4000, N.FLOAT32)
    assert need > 0
    assert call(M=4000, dt=N.FLOAT32) == N.ERR_ARG and b"workspace" in N.lib.nkl_last_error()
    assert call(M=4000, dt=N.FLOAT32, ws=FAKE, wsb=need - 1) == N.ERR_ARG
    assert call(M=4000, dt=N.FLOAT32, ws=ctypes.c_void_p(4096 + 16), wsb=need) == N.ERR_ALIGN
    assert call(B=0, q=None) == N.OK
    assert call(T=0, q=None) == N.OK


def test_sample_refusals(N):
    def call(**kw):
        a = dict(x=FAKE, stride=100, u=FAKE, ts=None, ks=None, ps=None, ms=None, t=1.0, k=0, p=1.0, m=0.0, token=FAKE, prob=FAKE,
                 B=2, V=100, dt=N.FLOAT32)
        assert not set(kw) - set(a)
        a.update(kw)
        return N.lib.nkl_sample(*a.values(), None)

    assert call(dt=3) == N.ERR_DTYPE
    for kw in (dict(V=0), dict(V=N.MAX_VOCAB + 1), dict(B=-1), dict(stride=-1)):
        assert call(**kw) == N.ERR_SHAPE
    for name in ("x", "u", "token", "prob"):
        assert call(**{name: None}) == N.ERR_ARG
    assert call(x=ctypes.c_void_p(4098)) == N.ERR_ALIGN
    assert call(B=0, x=None) == N.OK


def test_sample_numbers_out_of_range():
    import torch

    from nkilab import ops

    x, u = torch.empty(2, 10, device="meta"), torch.empty(2, device="meta")
    assert [tuple(t.shape) for t in ops.sample(x, u, 0.5, 3, 0.9, 0.1)] == [(2,), (2,)]
    for kw in (dict(temperature=-1.0), dict(temperature=math.nan), dict(top_k=-1), dict(top_p=1.1), dict(top_p=-0.1), dict(min_p=2.0)):
        with pytest.raises(ValueError):
            ops.sample(x, u, **kw)
    with pytest.raises(NotImplementedError):
        ops.sample(torch.zeros(2, 10), torch.zeros(2))


def test_page_operations_need_the_scales_of_a_cache_in_8_bits():
    import torch

    from nkilab import ops

    def m(*shape, dtype=torch.int32):
        return torch.empty(shape, dtype=dtype, device="meta")

    e4m3, e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    tables, lens, refs = m(3, 4), m(3), m(20)
    for lead in ((), (2,)):
        c, s = m(*lead, 20, 2, 16, 64, dtype=e4m3), m(*lead, 20, 2, 2, dtype=e8m0)
        plain = m(*lead, 20, 2, 16, 64, dtype=torch.bfloat16)
        for call in (lambda kc, ks, vs: ops.cache_fork(kc, kc, tables, lens, refs, m(1), m(1), ks, vs),
                     lambda kc, ks, vs: ops.cache_compact(kc, kc, tables, refs, ks, vs)):
            assert call(c, s, s)[0].shape == (3, 4) and call(plain, None, None)[0].shape == (3, 4)
            with pytest.raises(ValueError):
                call(c, s, None)
            with pytest.raises(ValueError):
                call(c, None, s)
            with pytest.raises(TypeError):
                call(c, None, None)
            with pytest.raises(TypeError):
                call(plain, s, s)


def test_page_operations_of_8_bits_refusals(N):
    nf, nc = N.lib.nkl_cache_fork_workspace_size(4, 3), N.lib.nkl_cache_compact_workspace_size(10)

    def fork(**kw):
        a = dict(kc=FAKE, vc=FAKE, cs=None, ks=FAKE, vs=FAKE, tables=FAKE, lens=FAKE, refs=FAKE, src=FAKE, dst=FAKE, to=FAKE,
                 lo=FAKE, ro=FAKE, missing=FAKE, ws=FAKE, wsb=nf, F=3, L=1, B=4, Hkv=2, d=64, P=10, page=16, M=4, block=8)
        assert not set(kw) - set(a)
        a.update(kw)
        return N.lib.nkl_cache_fork_8bit(*a.values(), None)

    def compact(**kw):
        a = dict(kc=FAKE, vc=FAKE, cs=None, ks=FAKE, vs=FAKE, tables=FAKE, refs=FAKE, to=FAKE, ro=FAKE, ws=FAKE, wsb=nc, L=1,
                 B=4, Hkv=2, d=64, P=10, page=16, M=4, block=8)
        assert not set(kw) - set(a)
        a.update(kw)
        return N.lib.nkl_cache_compact_8bit(*a.values(), None)

    for call in (fork, compact):
        for kw in (dict(d=24), dict(d=0), dict(L=0), dict(Hkv=0), dict(P=0), dict(page=0), dict(M=0), dict(block=0), dict(block=5),
                   dict(block=32), dict(B=-1)):
            assert call(**kw) == N.ERR_SHAPE
        for name in ("kc", "vc", "ks", "vs", "tables", "refs", "to", "ro", "ws"):
            assert call(**{name: None}) == N.ERR_ARG
        assert call(kc=ODD) == N.ERR_ALIGN and call(cs=strides(20480, 2048, 1024, 72)) == N.ERR_ALIGN
        assert call(wsb=0) == N.ERR_ARG
