"""Cases and plain forms of the decoding operators: attention for a tree of drafted tokens over a paged cache,
the cache's page operations, and the verification of drafted tokens.

``run`` computes an operator in plain torch (``own`` false) or through ``nkilab.ops`` (``own`` true) on the
state that ``prepare`` makes from a seed. ``exact`` gives the same results from the definitions in 64 bits.
"""
from __future__ import annotations

import functools
import math
import os
import sys

import numpy as np
import torch

own = False

ONE = 1 << 31  # probabilities and uniform numbers are whole multiples of 2^-31


@functools.lru_cache(None)
def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nki-kernel-lab_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from nkilab import ops

    return ops


_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# --------------------------------------------------------------------------- cases

def _attn(name, B, T, H, Hkv, d, page, ctx, dtype, tree):
    return dict(name=name, op="attention", B=B, T=T, H=H, Hkv=Hkv, d=d, page=page, ctx=ctx, dtype=dtype, tree=tree)


def _fork(name, L, B, F, Hkv, d, page, ctx, dtype):
    return dict(name=name, op="fork", L=L, B=B, F=F, Hkv=Hkv, d=d, page=page, ctx=ctx, dtype=dtype)


def _evict(name, L, B, F, Hkv, d, page, ctx, dtype):
    return dict(name=name, op="evict", L=L, B=B, F=F, Hkv=Hkv, d=d, page=page, ctx=ctx, dtype=dtype)


def _append(name, L, B, T, Hkv, d, page, ctx, dtype, picked):
    return dict(name=name, op="append", L=L, B=B, T=T, Hkv=Hkv, d=d, page=page, ctx=ctx, dtype=dtype, picked=picked)


def _verify(name, B, T, V, dtype, ratio):
    return dict(name=name, op="verify", B=B, T=T, V=V, dtype=dtype, ratio=ratio)


def listed():
    return [
        # one new token of one short conversation: the smallest call of a decoding loop, where latency counts
        _attn("attention 1 token", 1, 1, 32, 8, 128, 16, 203, "bf16", False),
        # four sequences of the decoder block's heads at its prompt length, 16 drafted tokens each
        _attn("attention 4x4096 mha", 4, 16, 32, 32, 128, 64, 4096, "bf16", True),
        # two long documents, a full tree of 64 drafted tokens, shared key/value heads
        _attn("attention 2x65536 gqa", 2, 64, 32, 8, 128, 64, 65536, "bf16", True),
        # fp32, short heads, pages that do not divide a tile, odd counts
        _attn("attention f32 odd", 5, 7, 8, 4, 64, 24, 1999, "f32", True),
        # two beams split off in a small model
        _fork("fork 2", 2, 8, 2, 8, 128, 16, 150, "bf16"),
        # a wide beam or many samples of shared prompts, a whole model's layers
        _fork("fork 64", 16, 96, 64, 8, 128, 64, 300, "bf16"),
        # one of four conversations ends in a small cache
        _evict("evict 1 of 4", 1, 4, 1, 8, 128, 16, 400, "bf16"),
        # every second conversation of a full cache ends
        _evict("evict 64 of 128", 8, 128, 64, 8, 128, 16, 500, "bf16"),
        # the accepted path of one conversation's tree, a small model
        _append("append path 1", 4, 1, 24, 8, 128, 16, 500, "bf16", True),
        # four prompts of the decoder block's configuration go to the cache
        _append("append prompt 4x4096", 1, 4, 4096, 32, 128, 64, 0, "bf16", False),
        # one conversation's tree
        _verify("verify tree 1x24", 1, 24, 32768, "f32", False),
        # a serving batch with chains drawn from a draft model's probabilities
        _verify("verify chain 64x8", 64, 8, 131072, "f32", True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "attention", "fork", "evict", "append", "verify"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    heads = [(8, 8), (8, 1), (32, 32), (32, 8), (12, 4), (8, 2)]
    if op == "attention":
        H, Hkv = rng.choice(heads)
        d = rng.choice([64, 128, 128])
        B, T = _log(rng, 1, 24), _log(rng, 1, 96)
        most = 2 * 65536 * 8 * 128 // (B * Hkv * d)
        most = min(most, 2 * 65536 * 64 * 32 * 128 // (B * T * H * d))
        if dtype == "f32":
            most = min(most, 8192, (1 << 28) // (B * T * H * d) + 1)
        ctx = _log(rng, 1, max(2, min(65536, most)))
        return _draw(_attn("", B, T, H, Hkv, d, rng.choice([8, 16, 24, 32, 64, 64, 128, 256]), ctx, dtype, rng.random() < 0.7))
    if op in ("fork", "evict"):
        Hkv, d, page = rng.choice([1, 2, 8, 32]), rng.choice([64, 128]), rng.choice([8, 16, 24, 64, 128])
        B = _log(rng, 2, 128)
        F = rng.randint(1, max(1, B // 2))
        ctx = _log(rng, page // 2, 600)
        row = 2 * Hkv * d * (2 if dtype == "bf16" else 4)
        L = _log(rng, 1, max(1, min(16, int(1.6e9) // (row * B * (ctx + page)))))
        return _draw((_fork if op == "fork" else _evict)("", L, B, F, Hkv, d, page, ctx, dtype))
    if op == "append":
        Hkv, d, page = rng.choice([1, 2, 8, 32]), rng.choice([64, 128]), rng.choice([8, 16, 24, 64, 128])
        picked = rng.random() < 0.6
        B = _log(rng, 1, 64 if picked else 8)
        T = _log(rng, 1, 96 if picked else 4096)
        row = 2 * Hkv * d * (2 if dtype == "bf16" else 4)
        T = max(1, min(T, 16384 * 16384 // (row * B)))
        ctx = _log(rng, 1, 500)
        L = _log(rng, 1, max(1, min(16, int(2.5e8) // (row * B * T))))
        return _draw(_append("", L, B, T, Hkv, d, page, ctx, dtype, picked))
    ratio = rng.random() < 0.5
    B, V = _log(rng, 1, 64), _log(rng, 500, 131072)
    T = _log(rng, 1, max(1, min(96, (1 << 27) // (B * V * (2 if ratio else 1)))))
    return _draw(_verify("", B, T, V, dtype, ratio))


def _draw(case):
    del case["name"]
    return case


# --------------------------------------------------------------------------- inputs

def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed), np.random.RandomState(seed % (1 << 32))


def _lens(case, r, count):
    """Lengths between half of the context and all of it; the first has all, of three or more the last is new."""
    ctx = case["ctx"]
    n = r.randint(ctx // 2, ctx + 1, count) if ctx > 1 else np.full(count, ctx)
    n[0] = ctx
    if count > 2 and case["op"] == "attention":
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


def _pool(case, g, r, lens, M, P, layers):
    """Pages in a scattered order: a table of [B, M], and the caches' k and v."""
    page, B = case["page"], len(lens)
    used = -(-lens // page)
    order, table, at = r.permutation(P), np.full((B, M), -1, np.int64), 0
    for b in range(B):
        table[b, :used[b]] = order[at:at + used[b]]
        at += used[b]
    shape = (*layers, P, case["Hkv"], page, case["d"])
    k, v = (torch.randn(shape, generator=g, device="cuda", dtype=_DTYPES[case["dtype"]]) for _ in range(2))
    return torch.from_numpy(table).int().cuda(), k, v


def _refs(table, P):
    refs = torch.zeros(P + 1, dtype=torch.int32, device="cuda")
    at = torch.where(table < 0, P, table).flatten().long()
    return refs.scatter_add_(0, at, torch.ones_like(at, dtype=torch.int32))[:P].contiguous()


def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x)).int().cuda()


def prepare(case, seed):
    g, r = _rng(seed)
    s = dict(case=case, op=case["op"])
    dt = _DTYPES[case["dtype"]]
    if case["op"] == "verify":
        B, T, V = case["B"], case["T"], case["V"]
        logits = torch.randn(B, T + 1, V, generator=g, device="cuda") * 2.5
        s["probs"] = logits.softmax(-1).to(dt)
        u = torch.rand(B, T + 1, generator=g, device="cuda")
        s["uniforms"] = u
        if case["ratio"]:
            q = logits[:, :T] + 0.5 * torch.randn(B, T, V, generator=g, device="cuda")
            s["draft_probs"] = q.softmax(-1).to(dt)
            tokens = _draws(s["draft_probs"].float(), torch.rand(B, T, generator=g, device="cuda"))
            s["parents"] = None
        else:
            # a tree of likely tokens: each token is one of its parent's row's best
            parents = _trees(r, B, T)
            top = s["probs"].float().topk(min(8, V), -1).indices.cpu().numpy()
            seen, toks = {}, np.zeros((B, T), np.int64)
            for b in range(B):
                for i in range(T):
                    key = (b, parents[b, i])
                    toks[b, i] = top[b, max(parents[b, i], -1) + 1, seen.get(key, 0) % top.shape[2]]
                    seen[key] = seen.get(key, 0) + 1
            tokens = torch.from_numpy(toks).cuda()
            s["draft_probs"], s["parents"] = None, _ints(parents)
        s["tokens"] = tokens.int()
        return s
    B, Hkv, d, page = case["B"], case["Hkv"], case["d"], case["page"]
    if case["op"] == "attention":
        T, H = case["T"], case["H"]
        lens = _lens(case, r, B)
        M = -(-case["ctx"] // page) + 1
        P = B * (M - 1) + 3
        s["tables"], s["k_cache"], s["v_cache"] = _pool(case, g, r, lens, M, P, ())
        qkv = torch.randn(B, T, H + 2 * Hkv, d, generator=g, device="cuda", dtype=dt)  # a fused projection's output
        s["q"], s["k"], s["v"] = qkv.split([H, Hkv, Hkv], 2)
        s["lens"] = _ints(lens)
        s["parents"] = _ints(_trees(r, B, T)) if case["tree"] else None
    elif case["op"] == "append":
        L, T = case["L"], case["T"]
        lens = _lens(case, r, B)
        count = r.randint(0, min(T, 8) + 1, B) if case["picked"] else np.full(B, T)
        count[0] = max(1, count[0])
        M = -(-(case["ctx"] + (min(T, 8) if case["picked"] else T)) // page) + 1
        s["tables"], s["k_cache"], s["v_cache"] = _pool(case, g, r, lens + count, M, B * (M - 1) + 3, (L,))
        s["k"], s["v"] = (torch.randn(L, B, T, Hkv, d, generator=g, device="cuda", dtype=dt) for _ in range(2))
        s["lens"] = _ints(lens)
        if case["picked"]:
            path = np.full((B, T), -1, np.int64)
            for b in range(B):
                path[b, :count[b]] = np.sort(r.choice(T, count[b], replace=False))
            s["path"], s["count"] = _ints(path), _ints(count)
        else:
            s["path"] = s["count"] = None
    else:
        L, F = case["L"], case["F"]
        live = B if case["op"] == "evict" else max(1, B - F)
        lens = np.zeros(B, np.int64)
        slots = r.permutation(B)
        lens[slots[:live]] = _lens(case, r, live)
        M = -(-case["ctx"] // page) + 1
        P = live * (M - 1) + F + 5
        s["tables"], s["k_cache"], s["v_cache"] = _pool(case, g, r, lens, M, P, (L,))
        s["lens"] = _ints(lens)
        s["refs"] = _refs(s["tables"], P)
        if case["op"] == "fork":
            s["src"], s["dst"] = _ints(slots[:live][r.randint(0, live, F)]), _ints(slots[B - F:])
        else:
            s["slots"] = _ints(np.sort(r.choice(B, F, replace=False)))
    return s


def _draws(p, u):
    """A token of each row by inverse distribution, for the inputs only."""
    return (p.cumsum(-1) <= (u * p.sum(-1))[..., None]).sum(-1).clamp(max=p.shape[-1] - 1)


# --------------------------------------------------------------------------- one pass

def run(s):
    op = s["op"]
    if own:
        ops = _ops()
        if op == "attention":
            return ops.attention_tree(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["parents"])
        if op == "append":
            lens = ops.cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["path"], s["count"])
            return dict(lens=lens, k=s["k_cache"], v=s["v_cache"])
        if op == "fork":
            tables, lens, refs, short = ops.cache_fork(s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["refs"], s["src"], s["dst"])
            return dict(tables=tables, lens=lens, refs=refs, short=short, k=s["k_cache"], v=s["v_cache"])
        if op == "evict":
            tables, lens, refs = ops.cache_free(s["tables"], s["lens"], s["refs"], s["slots"])
            tables, refs = ops.cache_compact(s["k_cache"], s["v_cache"], tables, refs)
            return dict(tables=tables, lens=lens, refs=refs, k=s["k_cache"], v=s["v_cache"])
        path, count, token = ops.verify_drafts(s["probs"], s["tokens"], s["uniforms"], s["parents"], s["draft_probs"])
        return dict(path=path, count=count, token=token)
    if op == "attention":
        return _plain_attention(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["parents"])
    if op == "append":
        return _plain_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["path"], s["count"])
    if op == "fork":
        return _plain_fork(s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["refs"], s["src"], s["dst"])
    if op == "evict":
        return _plain_evict(s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["refs"], s["slots"])
    return _plain_verify(s["probs"], s["tokens"], s["uniforms"], s["parents"], s["draft_probs"])


# --------------------------------------------------------------------------- plain forms

def _ancestors(parents):
    """[B, T, T]: whether j is i or an ancestor of i, for present tokens i."""
    B, T = parents.shape
    at = torch.arange(T, device=parents.device)
    present = parents >= -1
    up = torch.where(present, parents, -1).long()
    link = (up[:, :, None] == at) & present[:, None, :]
    reach = (link | torch.eye(T, dtype=torch.bool, device=parents.device)).float()
    for _ in range(max(1, (T - 1).bit_length())):  # paths of twice the length
        reach = (reach @ reach > 0).float()
    return (reach > 0) & present[:, :, None]


def _plain_attention(q, k, v, k_cache, v_cache, tables, lens, parents):
    B, T, H, d = q.shape
    P, Hkv, page, _ = k_cache.shape
    n = tables.shape[1] * page
    at = tables.clamp(0, P - 1).long()
    ks, vs = (c[at].transpose(1, 2).reshape(B, Hkv, n, d).float() for c in (k_cache, v_cache))
    seen = torch.arange(n, device=q.device) < lens[:, None]
    ks, vs = (torch.where(seen[:, None, :, None], c, 0.0) for c in (ks, vs))
    if parents is None:
        tree = torch.ones(T, T, dtype=torch.bool, device=q.device).tril().expand(B, T, T)
    else:
        tree = _ancestors(parents)
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


def _plain_append(k, v, k_cache, v_cache, tables, lens, path, count):
    L, B, T, Hkv, d = k.shape
    page = k_cache.shape[3]
    j = torch.arange(T, device=k.device)
    if path is None:
        path, count = j.expand(B, T), torch.full_like(lens, T)
    b, j = torch.nonzero(j < count[:, None], as_tuple=True)
    row, pos = path[b, j].long(), (lens[b] + j).long()
    at, slot = tables[b, pos // page].long(), pos % page
    k_cache[:, at, :, slot] = k[:, b, row].transpose(0, 1)
    v_cache[:, at, :, slot] = v[:, b, row].transpose(0, 1)
    return dict(lens=lens + count, k=k_cache, v=v_cache)


def _plain_fork(k_cache, v_cache, tables, lens, refs, src, dst):
    page, M, F = k_cache.shape[3], tables.shape[1], src.numel()
    s, t = src.long(), dst.long()
    n = lens[s].long()
    full, rest = n // page, n % page
    need = rest > 0
    free = (refs == 0).cumsum(0)
    short = (need.sum() - free[-1]).clamp_min(0)
    rank = need.cumsum(0) - need.long()
    fresh = torch.searchsorted(free, rank + 1).clamp(max=refs.numel() - 1)
    cols = torch.arange(M, device=s.device)
    old, rows = tables[t], tables[s]
    rows = torch.where(cols < full[:, None], rows, torch.where((cols == full[:, None]) & need[:, None], fresh[:, None].int(), -1))
    ok = short == 0
    new_tables, new_lens = tables.clone(), lens.clone()
    new_tables[t] = torch.where(ok, rows, old)
    new_lens[t] = torch.where(ok, n.int(), lens[t])
    pad = torch.cat([refs, refs.new_zeros(1)])
    for x, by in ((old, -1), (rows, 1)):
        pad.scatter_add_(0, torch.where((x >= 0) & ok, x, refs.numel()).flatten().long(), torch.full((x.numel(),), by, dtype=torch.int32, device=s.device))
    # the last page's used rows; a fork that needs no page writes a live page onto itself
    live = (refs > 0).int().argmax()
    come = torch.where(need, tables[s, full.clamp(max=M - 1)].long(), live)
    go = torch.where(need & ok, fresh, come)
    take = (torch.arange(page, device=s.device) < rest[:, None])[None, :, None, :, None]
    for c in (k_cache, v_cache):
        c[:, go] = torch.where(take, c[:, come], c[:, go])
    return dict(tables=new_tables, lens=new_lens, refs=pad[:-1], short=short.int().reshape(1), k=k_cache, v=v_cache)


def _plain_evict(k_cache, v_cache, tables, lens, refs, slots):
    at, P = slots.long(), refs.numel()
    gone = tables[at]
    pad = torch.cat([refs, refs.new_zeros(1)])
    pad.scatter_add_(0, torch.where(gone >= 0, gone, P).flatten().long(), torch.full((gone.numel(),), -1, dtype=torch.int32, device=refs.device))
    refs = pad[:-1]
    tables, lens = tables.clone(), lens.clone()
    tables[at], lens[at] = -1, 0
    live = refs > 0
    index = torch.arange(P, device=refs.device)
    low = index < live.sum()
    come, go = torch.nonzero(live & ~low).flatten(), torch.nonzero(~live & low).flatten()
    place = index.clone()
    place[come] = go
    for c in (k_cache, v_cache):
        c[:, go] = c[:, come]
    new_refs = torch.zeros_like(refs)
    new_refs[place[live]] = refs[live]
    tables = torch.where(tables >= 0, place[tables.clamp_min(0).long()].int(), -1)
    return dict(tables=tables, lens=lens, refs=new_refs, k=k_cache, v=v_cache)


def _whole(p):
    return (torch.nan_to_num(p.float(), nan=0.0).clamp(0, 1) * ONE).to(torch.int64)


def _plain_verify(probs, tokens, uniforms, parents, draft_probs):
    B, T = tokens.shape
    V = probs.shape[-1]
    at = torch.arange(T, device=probs.device)
    slot = torch.arange(B, device=probs.device)
    u = (uniforms.clamp(0, 1) * ONE).to(torch.int64).clamp(max=ONE - 1)
    good = (tokens >= 0) & (tokens < V)
    x = torch.where(good, tokens, 0).long()
    if draft_probs is not None or parents is None:
        up = (at - 1).expand(B, T)
        present = good
        ancestors = torch.ones(T, T, dtype=torch.bool, device=probs.device).tril().expand(B, T, T)
        brother = torch.zeros(B, T, T, dtype=torch.bool, device=probs.device)
    else:
        present = good & (parents >= -1)
        up = parents.long()
        ancestors = _ancestors(parents)
        brother = (up[:, :, None] == up[:, None, :]) & present[:, :, None] & present[:, None, :] & (at[:, None] > at)
    row = (up + 1).clamp(0, T)
    mine = torch.where(present, _whole(probs[slot[:, None], row, x]), 0)
    if draft_probs is not None:
        accept = u[:, :T] * _whole(draft_probs[slot[:, None], at, x]) < mine * ONE
    else:
        same = brother & (x[:, :, None] == x[:, None, :])
        mine = torch.where(same.any(-1), 0, mine)
        left = (ONE - (brother * mine[:, None, :]).sum(-1)).clamp_min(0)
        accept = u[:, :T] * left < mine * ONE
    accept &= present
    accept &= ~(brother & accept[:, None, :]).any(-1)
    on = accept & (~ancestors | accept[:, None, :]).all(-1)
    count = on.sum(-1)
    path = torch.where(on, at, T).sort(-1).values
    last = torch.where(on, at, -1).amax(-1)
    path = torch.where(path < T, path, -1)
    w = _whole(probs[slot, last + 1])
    whole = w
    if draft_probs is not None:
        stop = (last + 1).clamp(max=T - 1)
        out = _whole(draft_probs[slot, stop])
        w = torch.where(((last + 1 < T) & good[slot, stop])[:, None], (w - out).clamp_min(0), w)
    else:
        child = present & (up == last[:, None])
        w = torch.cat([w, w.new_zeros(B, 1)], 1).scatter(1, torch.where(child, x, V), 0)[:, :V]
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, whole)
    sums = w.cumsum(-1)
    total, last_u = sums[:, -1], u[:, T]
    t = (total >> 31) * last_u + (((total & (ONE - 1)) * last_u) >> 31)
    token = torch.where(total > 0, (sums <= t[:, None]).sum(-1), -1)
    return dict(path=path.int(), count=count.int(), token=token.int())


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    r = np.random.RandomState(1)  # the lengths of one seed
    if case["op"] == "verify":
        B, T, V = case["B"], case["T"], case["V"]
        rows = 2 if case["ratio"] else 1
        return dict(bytes=B * (V * rows * e + T * (16 + 2 * e)), flops=B * V * rows)
    B, Hkv, d, page = case["B"], case["Hkv"], case["d"], case["page"]
    row = 2 * Hkv * d * e  # k and v of one position
    if case["op"] == "attention":
        T, H = case["T"], case["H"]
        n = float(_lens(case, r, B).sum())
        return dict(bytes=(n + B * T) * row + 2 * B * T * H * d * e + 4 * n / page, flops=4.0 * d * H * T * (n + B * min(T, 8) / 2))
    if case["op"] == "append":
        count = B * (min(case["T"], 8) / 2 if case["picked"] else case["T"])
        return dict(bytes=2 * case["L"] * row * count, flops=0)
    if case["op"] == "fork":
        n = _lens(case, r, max(1, B - case["F"]))
        return dict(bytes=2 * case["L"] * row * case["F"] * float(np.mean(n % page)) + 8 * B * (-(-case["ctx"] // page) + 1), flops=0)
    n = -(-_lens(case, r, B) // page)
    pages, left = float(B * n.max()) + case["F"] + 5, float(n.sum()) * (B - case["F"]) / B
    moved = left * (pages - left) / pages
    return dict(bytes=2 * case["L"] * row * page * moved + 8 * B * (-(-case["ctx"] // page) + 1), flops=0)


# --------------------------------------------------------------------------- in 64 bits, from the definitions

def exact(case, seed):
    s = prepare(case, seed)
    return dict(attention=_exact_attention, append=_exact_append, fork=_exact_fork, evict=_exact_evict, verify=_exact_verify)[case["op"]](s)


def _exact_attention(s):
    c = s["case"]
    B, T, H, Hkv, d, page = (c[x] for x in ("B", "T", "H", "Hkv", "d", "page"))
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
            ks = torch.cat([s["k_cache"][pages, h].reshape(-1, d)[:n], s["k"][b, :, h]]).double()
            vs = torch.cat([s["v_cache"][pages, h].reshape(-1, d)[:n], s["v"][b, :, h]]).double()
            for g in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                w = (s["q"][b, :, g].double() @ ks.T / math.sqrt(d)).masked_fill(~see, -math.inf)
                out[b, here, g] = (w.softmax(-1) @ vs)[here]
    return out


def _small(s):
    return s["k_cache"].numel() < 1 << 26


def _exact_append(s):
    if not _small(s):
        return None
    k, v, kc, vc = (s[x].double() for x in ("k", "v", "k_cache", "v_cache"))
    lens, tables, page = s["lens"].tolist(), s["tables"].tolist(), kc.shape[3]
    counts = s["count"].tolist() if s["count"] is not None else [k.shape[2]] * len(lens)
    for b, n in enumerate(lens):
        for j in range(counts[b]):
            row = int(s["path"][b, j]) if s["path"] is not None else j
            at, slot = tables[b][(n + j) // page], (n + j) % page
            kc[:, at, :, slot], vc[:, at, :, slot] = k[:, b, row], v[:, b, row]
    return dict(lens=torch.tensor([n + m for n, m in zip(lens, counts)]), k=kc, v=vc)


def _exact_fork(s):
    if not _small(s):
        return None
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    lens, tables, refs, page = s["lens"].tolist(), s["tables"].tolist(), s["refs"].tolist(), kc.shape[3]
    M = len(tables[0])
    free = [p for p, n in enumerate(refs) if n == 0]
    forks = list(zip(s["src"].tolist(), s["dst"].tolist()))
    short = max(0, sum(lens[a] % page > 0 for a, _ in forks) - len(free))
    new_tables, new_lens = [list(t) for t in tables], list(lens)
    for a, b in forks if not short else []:
        for p in tables[b]:
            if p >= 0:
                refs[p] -= 1
        full, rest = divmod(lens[a], page)
        row = tables[a][:full]
        for p in row:
            refs[p] += 1
        if rest:
            p = free.pop(0)
            refs[p] += 1
            kc[:, p, :, :rest], vc[:, p, :, :rest] = kc[:, tables[a][full], :, :rest], vc[:, tables[a][full], :, :rest]
            row = row + [p]
        new_tables[b], new_lens[b] = row + [-1] * (M - len(row)), lens[a]
    return dict(tables=torch.tensor(new_tables), lens=torch.tensor(new_lens), refs=torch.tensor(refs), short=torch.tensor([short]), k=kc, v=vc)


def _exact_evict(s):
    if not _small(s):
        return None
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    lens, tables, refs = s["lens"].tolist(), s["tables"].tolist(), s["refs"].tolist()
    for b in s["slots"].tolist():
        for p in tables[b]:
            if p >= 0:
                refs[p] -= 1
        tables[b], lens[b] = [-1] * len(tables[b]), 0
    n = sum(x > 0 for x in refs)
    holes, place = [p for p in range(n) if refs[p] <= 0], list(range(len(refs)))
    for p in range(n, len(refs)):
        if refs[p] > 0:
            h = holes.pop(0)
            kc[:, h], vc[:, h] = kc[:, p], vc[:, p]
            refs[h], refs[p], place[p] = refs[p], 0, h
    tables = [[place[x] if x >= 0 else x for x in t] for t in tables]
    return dict(tables=torch.tensor(tables), lens=torch.tensor(lens), refs=torch.tensor(refs), k=kc, v=vc)


def _exact_verify(s):
    c = s["case"]
    B, T, V = c["B"], c["T"], c["V"]
    tokens, u = s["tokens"].tolist(), [[int(x * ONE) for x in r] for r in s["uniforms"].double().tolist()]
    parents = s["parents"].tolist() if s["parents"] is not None else [list(range(-1, T - 1))] * B
    row = lambda t, b, i: np.floor(t[b, i].double().cpu().numpy() * ONE).astype(object)  # noqa: E731
    paths, counts, nexts = [], [], []
    for b in range(B):
        at, path, p = -1, [], row(s["probs"], b, 0)
        left, w = ONE, p.copy()
        for i in range(T):
            if parents[b][i] != at or parents[b][i] < -1 or tokens[b][i] < 0:
                continue
            x = tokens[b][i]
            if s["draft_probs"] is not None:
                q = row(s["draft_probs"], b, i)
                take = u[b][i] * q[x] < p[x] * ONE
                w = w if take else np.maximum(p - q, 0)
            else:
                take = u[b][i] * max(left, 0) < w[x] * ONE
                left, w[x] = left - w[x], 0
            if take:
                at = i
                path.append(i)
                p = row(s["probs"], b, i + 1)
                left, w = ONE, p.copy()
        if not w.sum():
            w = p
        sums = np.cumsum(w)
        paths.append(path + [-1] * (T - len(path)))
        counts.append(len(path))
        nexts.append(int((sums <= u[b][T] * sums[-1] // ONE).sum()) if sums[-1] else -1)
    return dict(path=torch.tensor(paths), count=torch.tensor(counts), token=torch.tensor(nexts))
