"""Decoding with a paged key/value cache: the decoder block of nkilab.model run on a few new
tokens at a time, drafted tokens verified, accepted ones kept.

    cache = PagedCache(layers, slots, pages, kv_heads, head_dim)
    cache.reserve(extra)                          # pages for the tokens to come
    y, k, v = decode(blocks, x, cache)            # x [B, T, d_model]: a prompt's chunk, or drafts
    cache.append(k, v)                            # keep all of them, or an accepted path
    speculative_step(blocks, embedding, head, cache, last, drafts, uniforms, parents)

The reference computes whole prompts only (nkilab/model.py:70-89); everything here extends
it. All bookkeeping stays on the GPU: a step makes no host round trip, so it can be captured
in a CUDA graph (``PagedCache`` then keeps its tables in the same arrays, see ``_keep``).
"""
from __future__ import annotations

import torch

from . import ops
from .model import DecoderBlock, device_weights


class PagedCache:
    """Keys and values of `slots` sequences in `pages` pages of `page_size` positions each.

    k, v [layers, pages, kv_heads, page_size, head_dim]; tables [slots, pages of a slot],
    lens [slots], refs [pages] and missing [1] as in nkilab.ops. `max_len` bounds a slot's
    positions (default: all pages). The caches' contents start undefined.
    """

    def __init__(self, layers: int, slots: int, pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 max_len: int | None = None, dtype: torch.dtype = torch.bfloat16, device=None):
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        width = pages if max_len is None else -(-max_len // page_size)
        if min(layers, slots, pages, kv_heads, head_dim, page_size, width) < 1:
            raise ValueError("sizes of a cache must be positive")
        self.page_size = page_size
        self.k, self.v = (torch.empty(layers, pages, kv_heads, page_size, head_dim, dtype=dtype, device=dev)
                          for _ in range(2))
        self.tables = torch.full((slots, width), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        self.missing = torch.zeros(1, dtype=torch.int32, device=dev)

    def _keep(self, **new) -> None:
        """The arrays stay where they are, so that a captured graph finds them on replay."""
        for name, t in new.items():
            getattr(self, name).copy_(t)

    def _slots(self, values) -> torch.Tensor:
        return torch.as_tensor(values, dtype=torch.int32).to(self.lens.device)

    def reserve(self, extra) -> torch.Tensor:
        """Pages for `extra` more positions (one number, or one per slot). Returns `missing`
        [1], on the GPU: over 0, the pages did not suffice and none was given out, so that slots
        may lack the pages of the tokens to come (append then drops what does not fit)."""
        if isinstance(extra, int):
            extra = torch.full_like(self.lens, extra)
        tables, refs, missing = ops.cache_reserve(self.tables, self.lens, self.refs, self._slots(extra), self.page_size)
        self._keep(tables=tables, refs=refs, missing=missing)
        return self.missing

    def append(self, k, v, path=None, count=None) -> None:
        """Keeps rows of k and v [layers, slots, T, kv_heads, head_dim]; see ops.cache_append. A slot
        keeps what its pages hold: its length ends with them, and the rows after that are dropped."""
        lens = ops.cache_append(k, v, self.k, self.v, self.tables, self.lens, path, count)
        room = (self.tables >= 0).sum(1, dtype=torch.int32) * self.page_size
        torch.minimum(lens, room, out=self.lens)

    def fork(self, src, dst) -> torch.Tensor:
        """Slots `dst` become copies of slots `src`; returns `missing` [1] as reserve does."""
        tables, lens, refs, missing = ops.cache_fork(self.k, self.v, self.tables, self.lens, self.refs,
                                                     self._slots(src), self._slots(dst))
        self._keep(tables=tables, lens=lens, refs=refs, missing=missing)
        return self.missing

    def free(self, slots) -> None:
        tables, lens, refs = ops.cache_free(self.tables, self.lens, self.refs, self._slots(slots))
        self._keep(tables=tables, lens=lens, refs=refs)

    def compact(self) -> None:
        tables, refs = ops.cache_compact(self.k, self.v, self.tables, self.refs)
        self._keep(tables=tables, refs=refs)

    def attention(self, layer: int, q, k, v, parents=None, scale=None) -> torch.Tensor:
        return ops.attention_tree(q, k, v, self.k[layer], self.v[layer], self.tables, self.lens, parents, scale)


def decode(blocks: list[DecoderBlock], x: torch.Tensor, cache: PagedCache, parents=None):
    """The blocks on new tokens x [slots, T, d_model] of every slot, T <= 128, after its cached
    positions: (output [slots, T, d_model], k, v [layers, slots, T, heads, head_dim]). The
    tokens are a tree (parents, see ops.attention_tree) or, without it, follow one another.
    Nothing is kept: append k and v, whole or the accepted path of them."""
    B, T, d = x.shape
    ks, vs = [], []
    for layer, block in enumerate(blocks):
        cfg = block.cfg
        w = device_weights(block, x.dtype, x.device)
        x2 = x.reshape(B * T, d)
        h = ops.rmsnorm(x2, w["norm1"], cfg.eps)
        q, k, v = ops.matmul(h, w["wqkv"]).view(B, T, 3, cfg.n_heads, cfg.head_dim).unbind(2)
        a = cache.attention(layer, q, k, v, parents)
        ks.append(k)
        vs.append(v)
        x2, h = torch.ops.nkilab.add_rmsnorm(x2.contiguous(), ops.matmul(a.view(B * T, d), w["wo"]), w["norm2"], cfg.eps)
        if "wgu" in w:
            act = torch.ops.nkilab.matmul_swiglu(h, w["wgu"])
        else:
            act = ops.swiglu(ops.matmul(h, w["wg"]), ops.matmul(h, w["wu"]))
        if x.dtype == torch.bfloat16:
            x = torch.ops.nkilab.matmul_residual(act, w["wd"], x2)
        else:
            x = x2 + ops.matmul(act, w["wd"])
        x = x.view(B, T, d)
    return x, torch.stack(ks), torch.stack(vs)


def probabilities(x: torch.Tensor, head: torch.Tensor) -> torch.Tensor:
    """softmax(x @ head) in fp32: x [..., d], head [d, V]; V a multiple of 8 for bf16."""
    x2 = x.reshape(-1, x.shape[-1])
    logits = torch.ops.nkilab.matmul_f32out(x2, head) if x.dtype == torch.bfloat16 else ops.matmul(x2, head)
    return ops.softmax(logits).view(*x.shape[:-1], head.shape[1])


def speculative_step(blocks: list[DecoderBlock], embedding: torch.Tensor, head: torch.Tensor, cache: PagedCache,
                     last: torch.Tensor, drafts: torch.Tensor, uniforms: torch.Tensor, parents=None, draft_probs=None):
    """One step of every slot: `last` [slots], its latest token (not in the cache yet), and
    `drafts` [slots, T] after it, T <= 127, go through the blocks as one tree; the accepted
    ones are kept in the cache, for which pages have to be reserved (T + 1 positions; where that
    left pages missing, a slot without the room loses accepted tokens: look at `missing` first).

    parents, draft_probs and uniforms [slots, T + 1] as in ops.verify_drafts; embedding
    [V, d_model], head [d_model, V]. Returns (path, count, token): the accepted drafts of each
    slot and the token after them, the next step's `last`.
    """
    tokens = torch.cat([last[:, None], drafts], 1).clamp(0, embedding.shape[0] - 1)
    if parents is None:
        tree = None
    else:  # `last` is the root: the others move up by one, absent ones stay absent, and one whose
        # parent is no earlier token follows `last`, as it does in the verification
        late = parents >= torch.arange(parents.shape[1], device=parents.device)
        up = torch.where(parents < -1, parents, (parents + 1).masked_fill(late, 0))
        tree = torch.cat([torch.full_like(parents[:, :1], -1), up], 1)
    y, k, v = decode(blocks, embedding[tokens.long()], cache, tree)
    path, count, token = ops.verify_drafts(probabilities(y, head), drafts, uniforms, parents, draft_probs)
    rows = torch.cat([torch.zeros_like(path[:, :1]), torch.where(path < 0, path, path + 1)], 1)
    cache.append(k, v, rows, count + 1)
    return path, count, token
