"""Cases and plain forms of the operators around a decoding step: rotary positions, keys and values appended to a
paged cache with the rotation on the way (in 16, 32 or 8 bits), attention over a cache held in 8 bits, and sampling.

``run`` computes an operator in plain torch (``own`` false) or through ``nkilab.ops`` (``own`` true) on the
state that ``prepare`` makes from a seed. ``exact`` gives the same results from the definitions in 64 bits.

An 8-bit cache holds e4m3 numbers with one power of two (e8m0) for each block of positions and head: the smallest
2^e, e >= -100, with which the block's largest magnitude is at most 448 * 2^e. A block that grows keeps its rows, and
where its power of two grows, they are rounded again.
"""
from __future__ import annotations

import functools
import math
import os
import sys

import numpy as np
import torch

own = False

ONE = 1 << 31  # weights, shares and uniform numbers are whole multiples of 2^-31
LOWEST = -100  # of the powers of two
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@functools.lru_cache(None)
def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nki-kernel-lab_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from nkilab import ops

    return ops


_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# --------------------------------------------------------------------------- cases

def _rotary(name, B, T, H, d, part, far, dtype, layout, tree, grad):
    return dict(name=name, op="rotary", B=B, T=T, H=H, d=d, part=part, far=far, dtype=dtype, layout=layout, tree=tree, grad=grad)


def _append(name, B, T, H, Hkv, d, page, block, ctx, dtype, layout, part):
    """block 0: the cache has the type of the rows."""
    return dict(name=name, op="append", B=B, T=T, H=H, Hkv=Hkv, d=d, page=page, block=block, ctx=ctx, dtype=dtype, layout=layout, part=part)


def _keep(name, L, B, T, Hkv, d, page, block, ctx, dtype):
    return dict(name=name, op="keep", L=L, B=B, T=T, Hkv=Hkv, d=d, page=page, block=block, ctx=ctx, dtype=dtype)


def _attn(name, B, T, H, Hkv, d, page, block, ctx, dtype, tree):
    return dict(name=name, op="attention", B=B, T=T, H=H, Hkv=Hkv, d=d, page=page, block=block, ctx=ctx, dtype=dtype, tree=tree)


def _sample(name, B, V, dtype, rows):
    return dict(name=name, op="sample", B=B, V=V, dtype=dtype, rows=rows)


def listed():
    return [
        # the queries and keys of one new token at a far position: the smallest call, once per layer and token
        _rotary("rotary 1 token", 1, 1, 40, 128, 128, 131072, "bf16", "half", False, False),
        # a part of odd heads, interleaved, for trees of drafted tokens in a small fp32 model
        _rotary("rotary f32 odd tree", 5, 23, 12, 80, 48, 8192, "f32", "interleaved", True, False),
        # queries and keys of four prompts of the decoder block's configuration, there and back
        _rotary("rotary training 4x4096", 4, 4096, 64, 128, 128, 4096, "bf16", "half", False, True),
        # one new token of each of 64 conversations goes to an 8-bit cache
        _append("append 8-bit 64x1", 64, 1, 32, 8, 128, 64, 16, 700, "bf16", "half", 128),
        # chunks of prompts behind what is cached, pages that end inside a chunk, a part of the head rotated
        _append("append bf16 odd", 3, 101, 12, 4, 64, 24, 0, 500, "bf16", "interleaved", 32),
        # four prompts of the decoder block's configuration go to an 8-bit cache
        _append("append 8-bit prompt 4x4096", 4, 4096, 32, 32, 128, 64, 16, 0, "bf16", "half", 128),
        # the accepted paths of drafted trees, a small model's layers
        _keep("keep 8-bit paths", 4, 8, 24, 8, 128, 64, 16, 500, "bf16"),
        # one new token of one short conversation: latency
        _attn("attention 1 token", 1, 1, 32, 8, 128, 16, 16, 203, "bf16", False),
        # one new token of a serving batch of long conversations: the cache's bytes
        _attn("attention 32x8192 gqa", 32, 1, 32, 8, 128, 64, 16, 8192, "bf16", False),
        # two long documents, a full tree of 64 drafted tokens, shared key/value heads
        _attn("attention 2x65536 tree", 2, 64, 32, 8, 128, 64, 16, 65536, "bf16", True),
        # the next token of one conversation
        _sample("sample 1x32768", 1, 32768, "f32", False),
        # the next tokens of a serving batch, each conversation with its own settings
        _sample("sample 64x131072", 64, 131072, "f32", True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "append", "append", "keep", "attention", "attention", "attention", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    e = 2 if dtype == "bf16" else 4
    heads = [(8, 8), (8, 1), (32, 32), (32, 8), (12, 4), (8, 2)]
    page, block = rng.choice([(8, 8), (16, 16), (16, 4), (24, 8), (24, 24), (32, 16), (64, 16), (64, 64), (64, 32), (128, 16), (256, 128)])
    layout = rng.choice(["half", "half", "interleaved"])
    d = rng.choice([64, 80, 128, 128])
    part = rng.choice([d, d, d // 2, 16])
    if op == "rotary":
        H = rng.choice([1, 5, 8, 12, 24, 40, 64])
        tree = rng.random() < 0.3
        B = _log(rng, 1, 64)
        T = _log(rng, 1, 96) if tree else _log(rng, 1, max(1, min(8192, 16384 * 64 * 128 * 2 // (B * H * d * e))))
        return _draw(_rotary("", B, T, H, d, part, _log(rng, 100, 1 << 20), dtype, layout, tree, not tree and rng.random() < 0.4))
    if op == "append":
        H, Hkv = rng.choice(heads)
        B = _log(rng, 1, 64)
        T = _log(rng, 1, max(1, min(4096, 16384 * 96 * 128 * 2 // (B * (H + 2 * Hkv) * d * e))))
        ctx = _log(rng, 1, max(1, min(2000, (1 << 27) // (B * Hkv * d))))
        return _draw(_append("", B, T, H, Hkv, d, page, rng.choice([block, block, 0]), ctx, dtype, layout, part))
    if op == "keep":
        B, T, Hkv = _log(rng, 1, 64), _log(rng, 1, 96), rng.choice([1, 2, 8, 32])
        ctx = _log(rng, 1, 500)
        L = _log(rng, 1, max(1, min(16, (1 << 27) // (B * (ctx + 2 * page) * Hkv * d), (1 << 27) // (B * T * Hkv * d))))
        return _draw(_keep("", L, B, T, Hkv, d, page, block, ctx, dtype))
    if op == "attention":
        H, Hkv = rng.choice(heads)
        B, T = _log(rng, 1, 32), _log(rng, 1, 96)
        most = min(2 * 65536 * 8 * 128 // (B * Hkv * d), 2 * 65536 * 64 * 32 * 128 // (B * T * H * d))
        if dtype == "f32":
            most = min(most, 8192, (1 << 28) // (B * T * H * d) + 1)
        return _draw(_attn("", B, T, H, Hkv, d, page, block, _log(rng, 1, max(2, min(65536, most))), dtype, rng.random() < 0.6))
    B = _log(rng, 1, 128)
    return _draw(_sample("", B, _log(rng, 500, min(262144, 64 * 131072 // B)), dtype, rng.random() < 0.5))


def _draw(case):
    del case["name"]
    return case


# --------------------------------------------------------------------------- inputs

def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed), np.random.RandomState(seed % (1 << 32))


def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x)).int().cuda()


def _lens(case, r, count):
    """Lengths between half of the context and all of it; the first has all, of three or more the last is new."""
    ctx = case["ctx"]
    n = r.randint(ctx // 2, ctx + 1, count) if ctx > 1 else np.full(count, ctx)
    n[0] = ctx
    if count > 2:
        n[-1] = 0
    return n.astype(np.int64)


def _trees(r, B, T):
    """Parents of drafted tokens in random trees, most tokens near the root, and a padded tail in odd slots."""
    parents = np.full((B, T), -1, np.int64)
    for b in range(B):
        for i in range(1, T):
            parents[b, i] = r.randint(-1, i) if r.rand() < 0.5 else r.randint(max(-1, i // 2 - 2), i // 2 + 1)
        if b % 2:
            parents[b, T - T // 4:] = -2
    return parents


def _freqs(case):
    """Radians per position, in 64 bits; far positions slow the low frequencies down to an eighth, the high ones stay."""
    i = torch.arange(case["part"] // 2, dtype=torch.float64)
    f = 10000.0 ** (-2 * i / case["part"])
    if case.get("far", 0) > 8192:
        slow = ((4096 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * (slow + (1 - slow) / 8)
    return f.cuda()


def _blocks(x, block):
    """Rows [..., rows, d] in 64 bits or 32 as e4m3 codes and the blocks' powers of two."""
    y = x.float().unflatten(-2, (-1, block))
    e = _power(y.abs().amax((-1, -2)))
    codes = (y * torch.exp2(-e.float())[..., None, None]).to(E4M3)
    return codes.flatten(-3, -2), torch.exp2(e.float()).to(E8M0)


def _power(top):
    """The smallest e with top <= 448 * 2^e, from the bits of a float32."""
    bits = top.view(torch.int32)
    return ((bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=LOWEST)


def _pool(case, g, r, lens, M, P, lead):
    """Pages in a scattered order: a table of [B, M], and k and v caches with their powers of two (None in 16 or 32 bits)."""
    page, B, block = case["page"], len(lens), case["block"]
    used = -(-lens // page)
    order, table, at = r.permutation(P), np.full((B, M), -1, np.int64), 0
    for b in range(B):
        table[b, :used[b]] = order[at:at + used[b]]
        at += used[b]
    out = []
    for _ in range(2):
        x = torch.randn((*lead, P, case["Hkv"], page, case["d"]), generator=g, device="cuda", dtype=_DTYPES[case["dtype"]])
        if block:  # heads and blocks of different sizes
            x *= torch.exp2(torch.randint(-2, 3, (*lead, P, case["Hkv"], page // block, 1), generator=g, device="cuda").to(x.dtype)).repeat_interleave(block, -2)
        out.append(_blocks(x, block) if block else (x, None))
    return _ints(table), out[0][0], out[1][0], out[0][1], out[1][1]


def prepare(case, seed):
    g, r = _rng(seed)
    op = case["op"]
    s = dict(case=case, op=op)
    dt = _DTYPES[case["dtype"]]
    B = case["B"]
    if op == "rotary":
        T, H, d = case["T"], case["H"], case["d"]
        x = torch.randn(B, T, H + 2, d, generator=g, device="cuda", dtype=dt)  # a fused projection's output, its values last
        s["x"] = x[:, :, :H] if not case["grad"] else x[:, :, :H].contiguous().requires_grad_()
        s["grad"] = torch.randn(B, T, H, d, generator=g, device="cuda", dtype=dt) if case["grad"] else None
        s["positions"] = _ints(r.randint(0, case["far"] + 1, B)) if not case["grad"] else _ints(np.tile(np.arange(T), (B, 1)))
        s["parents"] = _ints(_trees(r, B, T)) if case["tree"] else None
        s["freqs"], s["interleaved"] = _freqs(case), case["layout"] == "interleaved"
        return s
    if op == "sample":
        V = case["V"]
        s["logits"] = (torch.randn(B, V, generator=g, device="cuda") * 2.5).to(dt)
        if B > 2:  # a grammar leaves few tokens of the last row
            s["logits"][-1, torch.rand(V, generator=g, device="cuda") < 0.999] = -math.inf
        s["uniforms"] = torch.rand(B, generator=g, device="cuda")
        if case["rows"]:
            s["temperature"] = torch.from_numpy(r.choice([0.0, 0.6, 0.8, 1.0, 1.3], B).astype(np.float32)).cuda()
            s["top_k"] = _ints(r.choice([0, 0, 1, 40, 1000], B))
            s["top_p"] = torch.from_numpy(r.choice([1.0, 0.5, 0.9, 0.95], B).astype(np.float32)).cuda()
            s["min_p"] = torch.from_numpy(r.choice([0.0, 0.0, 0.02, 0.1], B).astype(np.float32)).cuda()
        else:
            s["temperature"], s["top_k"], s["top_p"], s["min_p"] = 0.8, 0, 0.95, 0.0
        return s
    T, Hkv, d, page, block = case["T"], case["Hkv"], case["d"], case["page"], case["block"]
    lens = _lens(case, r, B)
    s["lens"] = _ints(lens)
    if op == "attention":
        H, M = case["H"], -(-case["ctx"] // page) + 1
        s["tables"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"] = _pool(case, g, r, lens, M, B * (M - 1) + 3, ())
        s["q"], s["k"], s["v"] = torch.randn(B, T, H + 2 * Hkv, d, generator=g, device="cuda", dtype=dt).split([H, Hkv, Hkv], 2)
        s["parents"] = _ints(_trees(r, B, T)) if case["tree"] else None
    elif op == "append":
        H = case["H"]
        count = np.full(B, T)
        if B > 1:  # a padded batch
            count[-1] = r.randint(0, T + 1)
        M = -(-(case["ctx"] + T) // page) + 1
        s["tables"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"] = _pool(case, g, r, lens + count, M, B * (M - 1) + 3, ())
        s["q"], s["k"], s["v"] = torch.randn(B, T, H + 2 * Hkv, d, generator=g, device="cuda", dtype=dt).split([H, Hkv, Hkv], 2)
        s["count"] = _ints(count)
        s["freqs"], s["interleaved"] = _freqs(case), case["layout"] == "interleaved"
    else:
        L, most = case["L"], min(T, 8)
        count = r.randint(0, most + 1, B)
        count[0] = max(1, count[0])
        M = -(-(case["ctx"] + most) // page) + 1
        s["tables"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"] = _pool(case, g, r, lens + count, M, B * (M - 1) + 3, (L,))
        s["k"], s["v"] = (torch.randn(L, B, T, Hkv, d, generator=g, device="cuda", dtype=dt) for _ in range(2))
        path = np.full((B, T), -1, np.int64)
        for b in range(B):
            path[b, :count[b]] = np.sort(r.choice(T, count[b], replace=False))
        s["path"], s["count"] = _ints(path), _ints(count)
    return s


# --------------------------------------------------------------------------- one pass

def run(s):
    op = s["op"]
    if own:
        ops = _ops()
        if op == "rotary":
            y = ops.rotary(s["x"], s["positions"], s["freqs"], s["parents"], interleaved=s["interleaved"])
            return y if s["grad"] is None else (y, torch.autograd.grad(y, s["x"], s["grad"])[0])
        if op == "append":
            q, k = ops.rotary_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["freqs"], s["count"],
                                     interleaved=s["interleaved"], k_scales=s["k_scales"], v_scales=s["v_scales"])
            return _state(s, q=q, k=k)
        if op == "keep":
            lens = ops.cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["path"], s["count"], s["k_scales"], s["v_scales"])
            return _state(s, lens=lens)
        if op == "attention":
            return ops.attention_tree(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["parents"],
                                      k_scales=s["k_scales"], v_scales=s["v_scales"])
        token, prob = ops.sample(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        return dict(token=token, prob=prob)
    if op == "rotary":
        with torch.no_grad():
            at = _plain_positions(s["positions"], s["parents"], s["x"].shape[1])
            y = _plain_rotary(s["x"], at, s["freqs"], s["interleaved"])
            return y if s["grad"] is None else (y, _plain_rotary(s["grad"], at, -s["freqs"], s["interleaved"]))
    if op == "append":
        at = _plain_positions(s["lens"], None, s["q"].shape[1])
        k32 = _plain_rotary(s["k"], at, s["freqs"], s["interleaved"], torch.float32)
        _plain_keep(s, k32[None], s["v"][None], s["count"])
        return _state(s, q=_plain_rotary(s["q"], at, s["freqs"], s["interleaved"]), k=k32.to(s["k"].dtype))
    if op == "keep":
        at = s["path"].clamp_min(0).long()[None, :, :, None, None].expand_as(s["k"])
        _plain_keep(s, s["k"].gather(2, at), s["v"].gather(2, at), s["count"])
        return _state(s, lens=s["lens"] + s["count"])
    if op == "attention":
        return _plain_attention(s["q"], s["k"], s["v"], _plain_values(s["k_cache"], s["k_scales"]), _plain_values(s["v_cache"], s["v_scales"]), s["tables"], s["lens"], s["parents"])
    return _plain_sample(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


def _state(s, **more):
    more |= dict(k_cache=s["k_cache"], v_cache=s["v_cache"])
    return more if s["k_scales"] is None else more | dict(k_scales=s["k_scales"], v_scales=s["v_scales"])


# --------------------------------------------------------------------------- plain forms

def _links(parents):
    """[B, T, T]: whether j is i or an ancestor of i; [B, T]: whether a token is present."""
    B, T = parents.shape
    at = torch.arange(T, device=parents.device)
    present = parents >= -1
    up = torch.where(present, parents, -1).long()
    link = (up[:, :, None] == at) & present[:, None, :]
    reach = (link | torch.eye(T, dtype=torch.bool, device=parents.device)).float()
    for _ in range(max(1, (T - 1).bit_length())):  # paths of twice the length
        reach = (reach @ reach > 0).float()
    return reach > 0, present


def _plain_positions(start, parents, T):
    """[B, T]: the positions given, or each sequence's first one and a token's depth below it."""
    if start.dim() == 2:
        return start
    if parents is None:
        return start[:, None] + torch.arange(T, device=start.device)
    reach, present = _links(parents)
    return start[:, None] + torch.where(present, reach.sum(-1) - 1, 0)


def _plain_rotary(x, positions, freqs, interleaved, out=None):
    r = 2 * freqs.numel()
    angle = positions.double()[:, :, None, None] * freqs
    c, s = angle.cos().float(), angle.sin().float()
    y = x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., :r // 2], y[..., r // 2:r])
    a, b = a * c - b * s, b * c + a * s
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, y[..., r:]], -1).to(out or x.dtype)


def _plain_values(cache, scales):
    block = cache.shape[-2] // scales.shape[-1]
    return (cache.float().unflatten(-2, (-1, block)) * scales.float()[..., None, None]).flatten(-3, -2)


def _plain_keep(s, k, v, count):
    """Rows k and v [layers, B, T, heads, d], those before count[b], to the pages behind lens[b]."""
    lens, tables = s["lens"].long(), s["tables"]
    L, B, T, H, d = k.shape
    for rows, name in ((k, "k"), (v, "v")):
        cache = s[name + "_cache"].view(L, *s[name + "_cache"].shape[-4:])
        page = cache.shape[3]
        if s[name + "_scales"] is None:
            b, j = torch.nonzero(torch.arange(T, device=k.device) < count[:, None], as_tuple=True)
            pos = lens[b] + j
            cache[:, tables[b, pos // page].long(), :, pos % page] = rows[:, b, j].transpose(0, 1).to(cache.dtype)
            continue
        scales = s[name + "_scales"].view(L, *s[name + "_scales"].shape[-3:])
        block = page // scales.shape[-1]
        # the blocks that rows come to: [B, n, block] positions, of which some are old and some new
        n = (T + block - 2) // block + 1
        pos = (lens[:, None] // block + torch.arange(n, device=k.device))[:, :, None] * block + torch.arange(block, device=k.device)
        new = (pos >= lens[:, None, None]) & (pos < (lens + count)[:, None, None])
        old = pos < lens[:, None, None]
        b, i = torch.nonzero(new.any(-1), as_tuple=True)
        pos, new, old = pos[b, i], new[b, i], old[b, i]
        at, part, slot = tables[b, pos[:, 0] // page].long(), (pos[:, 0] % page) // block, pos % page
        was = _code(scales[:, at, :, part]).transpose(0, 1)  # [layers, blocks, heads]
        x = rows[:, b[:, None], (pos - lens[b, None]).clamp(0, T - 1)].float().transpose(2, 3)  # [layers, blocks, heads, block, d]
        x = torch.where(new[None, :, None, :, None], x, 0.0)
        e = _power(x.abs().amax((-1, -2)))
        e = torch.where(old.any(-1)[None, :, None], torch.maximum(e, was), e)
        codes = cache[:, at[:, None], :, slot].permute(2, 0, 3, 1, 4).float()
        codes = torch.where(new[None, :, None, :, None], x * torch.exp2(-e.float())[..., None, None], codes * torch.exp2((was - e).float().clamp(max=0))[..., None, None])
        keep = (new | old)[:, :, None, None, None]
        # a row that is neither stays: e4m3 values return to the bytes that they came from
        here = cache[:, at[:, None], :, slot].float()
        cache[:, at[:, None], :, slot] = torch.where(keep, codes.permute(1, 3, 0, 2, 4), here).to(E4M3)
        scales[:, at, :, part] = torch.exp2(e.float()).transpose(0, 1).to(E8M0)


def _code(scales):
    return scales.view(torch.uint8).int() - 127


def _plain_attention(q, k, v, k_cache, v_cache, tables, lens, parents):
    B, T, H, d = q.shape
    P, Hkv, page, _ = k_cache.shape
    n = tables.shape[1] * page
    at = tables.clamp(0, P - 1).long()
    ks, vs = (c[at].transpose(1, 2).reshape(B, Hkv, n, d) for c in (k_cache, v_cache))
    seen = torch.arange(n, device=q.device) < lens[:, None]
    ks, vs = (torch.where(seen[:, None, :, None], c, 0.0) for c in (ks, vs))
    if parents is None:
        tree = torch.ones(T, T, dtype=torch.bool, device=q.device).tril().expand(B, T, T)
    else:
        tree, present = _links(parents)
        tree = tree & present[:, :, None]
    mask = torch.cat([seen[:, None, :].expand(B, T, n) & tree.any(-1, keepdim=True), tree], -1)
    ks, vs = torch.cat([ks, k.transpose(1, 2).float()], 2), torch.cat([vs, v.transpose(1, 2).float()], 2)
    qs = q.float().reshape(B, T, Hkv, H // Hkv, d).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, d)
    w = (qs @ ks.transpose(-1, -2)).view(B, Hkv, H // Hkv, T, -1) / math.sqrt(d)
    w = w.masked_fill(~mask[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(top == -math.inf, 0.0, top))
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-30)
    out = w.view(B, Hkv, -1, w.shape[-1]) @ vs
    return out.view(B, Hkv, H // Hkv, T, d).permute(0, 3, 1, 2, 4).reshape(B, T, H, d).to(q.dtype)


def _plain_sample(logits, uniforms, temperature, top_k, top_p, min_p):
    B, V = logits.shape
    row = lambda x, t: (x if torch.is_tensor(x) else torch.full((B,), x, device=logits.device)).to(t)[:, None]  # noqa: E731
    t, k, p, low = row(temperature, torch.float64), row(top_k, torch.int64), row(top_p, torch.float64), row(min_p, torch.float64)
    x = torch.where(logits.isnan(), -math.inf, logits.double())
    top = x.amax(-1, keepdim=True)
    greedy = ~(t > 0)
    z = torch.where(x == top, 0.0, (x - top) / torch.where(greedy, 1.0, t))
    w = torch.where(x > -math.inf, (z.exp() * ONE).floor(), 0.0).long()
    order = x.sort(dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    place = torch.arange(V, device=x.device)
    k = torch.where(greedy, 1, torch.where(k > 0, k, V))
    ws = torch.where(place < k, ws, 0)
    before = ws.cumsum(-1) - ws
    share = torch.where(p < 1, (p.clamp(0, 1) * ONE).floor(), ONE).long()
    need = _share(ws.sum(-1, keepdim=True), share).clamp_min(1)
    keep = (place < k) & (before < need) & (ws >= low.clamp(0, 1) * ONE)
    w = torch.zeros_like(w).scatter(1, order, torch.where(keep, ws, 0))
    sums = w.cumsum(-1)
    total = sums[:, -1:]
    u = (uniforms.double()[:, None].clamp(0, 1) * ONE).long().clamp(max=ONE - 1)
    token = (sums <= _share(total, u)).sum(-1, keepdim=True)
    some = total > 0
    prob = w.gather(1, token.clamp(max=V - 1)).double() / total.clamp_min(1)
    return dict(token=torch.where(some, token, -1)[:, 0].int(), prob=torch.where(some, prob, 0.0)[:, 0].float())


def _share(total, share):
    """total * share / 2^31, rounded down."""
    return (total >> 31) * share + (((total & (ONE - 1)) * share) >> 31)


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    op, e = case["op"], 2 if case["dtype"] == "bf16" else 4
    r = np.random.RandomState(1)  # the lengths of one seed
    B = case["B"]
    if op == "sample":
        return dict(bytes=B * (case["V"] * e + 12), flops=4.0 * B * case["V"])
    T, d = case["T"], case["d"]
    if op == "rotary":
        n = B * T * case["H"] * d * (2 if case["grad"] else 1)
        return dict(bytes=2 * n * e + B * T * 4, flops=3.0 * n * case["part"] / d)
    Hkv, block = case["Hkv"], case["block"]
    c = 1 if block else e
    kept = 2 * Hkv * (d * c + (1 / block if block else 0))  # k and v of one cached position
    if op == "append":
        n, H = B * T, case["H"]
        return dict(bytes=n * ((2 * H + 3 * Hkv) * d * e + kept), flops=3.0 * n * (H + Hkv) * case["part"])
    if op == "keep":
        n = case["L"] * B * min(T, 8) / 2
        return dict(bytes=n * (2 * Hkv * d * e + kept), flops=0)
    n, H = float(_lens(case, r, B).sum()), case["H"]
    return dict(bytes=n * kept + B * T * (2 * H + 2 * Hkv) * d * e + 4 * n / case["page"], flops=4.0 * d * H * T * (n + B * min(T, 8) / 2))


# --------------------------------------------------------------------------- in 64 bits, from the definitions

def exact(case, seed):
    s = prepare(case, seed)
    return dict(rotary=_exact_rotary, append=_exact_append, keep=_exact_append, attention=_exact_attention, sample=_exact_sample)[case["op"]](s)


def _depths(parents):
    out = []
    for row in parents.tolist():
        depth = []
        for p in row:
            depth.append(depth[p] + 1 if p >= 0 and row[p] >= -1 else 0)
        out.append([0 if p < -1 else n for p, n in zip(row, depth)])
    return torch.tensor(out, device="cuda")


def _turned(x, positions, freqs, interleaved):
    """Pairs as complex numbers, turned."""
    r = 2 * freqs.numel()
    y = x.double()
    pairs = y[..., :r].unflatten(-1, (r // 2, 2)) if interleaved else y[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(freqs), positions.double()[..., None, None] * freqs)
    pairs = torch.view_as_real(z)
    return torch.cat([pairs.flatten(-2) if interleaved else pairs.transpose(-1, -2).flatten(-2), y[..., r:]], -1)


def _exact_rotary(s):
    c = s["case"]
    at = s["positions"]
    if at.dim() == 1:
        at = at[:, None] + (torch.arange(c["T"], device="cuda") if s["parents"] is None else _depths(s["parents"]))
    y = _turned(s["x"].detach(), at, s["freqs"], s["interleaved"])
    return y if s["grad"] is None else (y, _turned(s["grad"], -at, s["freqs"], s["interleaved"]))


def _exact_append(s):
    c = s["case"]
    lens, counts, block, page = s["lens"].tolist(), s["count"].tolist(), c["block"], c["page"]
    if c["B"] * max(counts) // max(block, 1) > 3000 * (1 if block else 10):
        return None  # one block after the other
    out = {}
    if c["op"] == "append":
        at = s["lens"][:, None] + torch.arange(c["T"], device="cuda")
        k, v = _turned(s["k"], at, s["freqs"], s["interleaved"]), s["v"].double()
        out["q"], out["k"] = _turned(s["q"], at, s["freqs"], s["interleaved"]), k
        rows = dict(k=k[None], v=v[None])
    else:
        rows = dict(k=s["k"].double(), v=s["v"].double())
        out["lens"] = torch.tensor([n + m for n, m in zip(lens, counts)])
    tables = s["tables"].tolist()
    for name in ("k", "v"):
        cache = s[name + "_cache"].double().view(-1, *s[name + "_cache"].shape[-4:])
        scales = s[name + "_scales"].double().view(cache.shape[0], *s[name + "_scales"].shape[-3:]) if block else None
        for b, n in enumerate(lens):
            row = list(range(counts[b])) if c["op"] == "append" else s["path"][b, :counts[b]].tolist()
            x = rows[name][:, b, row].transpose(1, 2)  # [layers, heads, rows, d]
            done = 0
            while done < counts[b]:
                at, step = n + done, block or 1
                p, slot = tables[b][at // page], at % page
                more = min(step - at % step, counts[b] - done)
                new = x[:, :, done:done + more]
                if block:
                    i, first = slot // block, slot - slot % block
                    e = torch.clamp(torch.ceil(torch.log2(new.abs().amax((-1, -2)) / 448)), min=LOWEST)
                    e = torch.where(448 * torch.exp2(e - 1) >= new.abs().amax((-1, -2)), torch.clamp(e - 1, min=LOWEST), e)
                    if slot > first:
                        e = torch.maximum(e, torch.log2(scales[:, p, :, i]).round())
                        old = cache[:, p, :, first:slot] * scales[:, p, :, i, None, None]
                        cache[:, p, :, first:slot] = _e4m3(old / torch.exp2(e)[..., None, None])
                    scales[:, p, :, i] = torch.exp2(e)
                    new = _e4m3(new / torch.exp2(e)[..., None, None])
                cache[:, p, :, slot:slot + more] = new
                done += more
        out[name + "_cache"] = cache.view(s[name + "_cache"].shape)
        if block:
            out[name + "_scales"] = scales.view(s[name + "_scales"].shape)
    return out


def _e4m3(x):
    """Four significant bits, the exponent at least -6, ties to even."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -20))).clamp(min=-6)
    return torch.round(x * torch.exp2(3 - e)) * torch.exp2(e - 3)


def _exact_attention(s):
    c = s["case"]
    B, T, H, Hkv, d, page, block = (c[x] for x in ("B", "T", "H", "Hkv", "d", "page", "block"))
    lens, tables = s["lens"].tolist(), s["tables"].long()
    parents = s["parents"].tolist() if s["parents"] is not None else [list(range(-1, T - 1))] * B
    out = torch.zeros(B, T, H, d, dtype=torch.float64, device="cuda")
    for b in range(B):
        n = lens[b]
        pages = tables[b, :-(-n // page)]
        see = torch.zeros(T, T, dtype=torch.bool)
        for i in range(T):
            if parents[b][i] >= -1:
                see[i, i] = True
                j = parents[b][i]
                while j >= 0 and parents[b][j] >= -1:
                    see[i, j] = True
                    j = parents[b][j]
        here = see.any(1).cuda()
        see = torch.cat([here[:, None].expand(T, n), see.cuda()], 1)
        for h in range(Hkv):
            ks, vs = (torch.cat([(s[x + "_cache"][pages, h].double() * s[x + "_scales"][pages, h].double().repeat_interleave(block, 1)[..., None]).reshape(-1, d)[:n],
                                 s[x][b, :, h].double()]) for x in ("k", "v"))
            for g in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                w = (s["q"][b, :, g].double() @ ks.T / math.sqrt(d)).masked_fill(~see, -math.inf)
                out[b, here, g] = (w.softmax(-1) @ vs)[here]
    return out


def _exact_sample(s):
    x = s["logits"].double().cpu().numpy()
    B, V = x.shape
    of = lambda v, b: float(v[b]) if torch.is_tensor(v) else v  # noqa: E731
    tokens, probs = [], []
    for b in range(B):
        t, k, p, low = (of(s[n], b) for n in ("temperature", "top_k", "top_p", "min_p"))
        order = np.lexsort((np.arange(V), -x[b]))
        order = order[np.isfinite(x[b][order])]
        if t == 0:
            order, t = order[:1], 1.0
        if k > 0:
            order = order[:int(k)]
        if not len(order):
            tokens.append(-1)
            probs.append(0.0)
            continue
        w = np.floor(np.exp((x[b][order] - x[b][order[0]]) / t) * ONE).astype(np.int64)
        if p < 1:
            need = max(1, int(w.sum()) * int(p * ONE) // ONE)
            w = w[:int((np.cumsum(w) < need).sum()) + 1]
        w = w[w >= low * ONE]
        order = order[:len(w)]
        back = np.argsort(order)
        sums = np.cumsum(w[back])
        at = back[int((sums <= int(sums[-1]) * int(float(s["uniforms"][b]) * ONE) // ONE).sum())]
        tokens.append(int(order[at]))
        probs.append(float(w[at]) / float(sums[-1]))
    return dict(token=torch.tensor(tokens), prob=torch.tensor(probs, dtype=torch.float64))
