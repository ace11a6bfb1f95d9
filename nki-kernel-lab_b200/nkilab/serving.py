"""Decoding with a paged key/value cache: the decoder block of nkilab.model run on a few new
tokens at a time, drafted tokens verified, accepted ones kept.

    cache = PagedCache(layers, slots, pages, kv_heads, head_dim)
    cache.reserve(extra)                          # pages for the tokens to come
    y, k, v = decode(blocks, x, cache)            # x [B, T, d_model]: a prompt's chunk, or drafts
    cache.append(k, v)                            # keep all of them, or an accepted path
    speculative_step(blocks, embedding, head, cache, last, drafts, uniforms, parents)

or, with rotary positions and sampling, on a cache of any kind,

    cache = PagedCache(layers, slots, pages, kv_heads, head_dim, dtype=torch.float8_e4m3fn)
    rotary = Rotary(head_dim, scaling="yarn", factor=4, trained=4096)
    y = extend(blocks, embedding[prompts], cache, rotary, count)
    token, prob = step(blocks, embedding, head, cache, last, uniforms, rotary, temperature=0.8, top_p=0.95)

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
    positions (default: all pages). The caches' contents start undefined. With dtype
    torch.float8_e4m3fn k and v are in 8 bits, with scales k_scales, v_scales [layers, pages, kv_heads,
    page_size / block], one for each `block` positions (see ops.cache_append).
    """

    def __init__(self, layers: int, slots: int, pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 max_len: int | None = None, dtype: torch.dtype = torch.bfloat16, device=None, block: int = 16):
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        width = pages if max_len is None else -(-max_len // page_size)
        if min(layers, slots, pages, kv_heads, head_dim, page_size, width) < 1:
            raise ValueError("sizes of a cache must be positive")
        self.page_size = page_size
        self.k, self.v = (torch.empty(layers, pages, kv_heads, page_size, head_dim, dtype=dtype, device=dev)
                          for _ in range(2))
        self.k_scales = self.v_scales = None
        if dtype == torch.float8_e4m3fn:
            if block < 1 or page_size % block:
                raise ValueError(f"blocks of {block} positions do not divide pages of {page_size}")
            shape = (layers, pages, kv_heads, page_size // block)
            self.k_scales, self.v_scales = (torch.full(shape, 127, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)
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
        self._grow(ops.cache_append(k, v, self.k, self.v, self.tables, self.lens, path, count, self.k_scales, self.v_scales))

    def _grow(self, lens) -> None:
        room = (self.tables >= 0).sum(1, dtype=torch.int32) * self.page_size
        torch.minimum(lens, room, out=self.lens)

    def fork(self, src, dst) -> torch.Tensor:
        """Slots `dst` become copies of slots `src`; returns `missing` [1] as reserve does."""
        tables, lens, refs, missing = ops.cache_fork(self.k, self.v, self.tables, self.lens, self.refs,
                                                     self._slots(src), self._slots(dst), self.k_scales, self.v_scales)
        self._keep(tables=tables, lens=lens, refs=refs, missing=missing)
        return self.missing

    def free(self, slots) -> None:
        tables, lens, refs = ops.cache_free(self.tables, self.lens, self.refs, self._slots(slots))
        self._keep(tables=tables, lens=lens, refs=refs)

    def compact(self) -> None:
        tables, refs = ops.cache_compact(self.k, self.v, self.tables, self.refs, self.k_scales, self.v_scales)
        self._keep(tables=tables, refs=refs)

    def _layer_scales(self, layer: int):
        return (None, None) if self.k_scales is None else (self.k_scales[layer], self.v_scales[layer])

    def attention(self, layer: int, q, k, v, parents=None, scale=None) -> torch.Tensor:
        return ops.attention_tree(q, k, v, self.k[layer], self.v[layer], self.tables, self.lens, parents, scale,
                                  *self._layer_scales(layer))

    def write(self, layer: int, q, k, v, rotary, count=None):
        """q and k turned to their positions, (q, k); k and v kept behind the slots' cached positions
        in this layer (see ops.rotary_append). The lengths are to follow when all layers have them."""
        return ops.rotary_append(q, k, v, self.k[layer], self.v[layer], self.tables, self.lens, rotary.freqs, count,
                                 rotary.interleaved, rotary.magnitude, *self._layer_scales(layer))


class Rotary:
    """Rotary positions of a model: `rotary_dim` entries of each head (default: all) turn with
    frequencies base^(-2i / rotary_dim), stretched for long contexts as ops.rotary_frequencies does. A model
    with frequencies of its own sets `freqs` (float64 on the GPU) and `magnitude`."""

    def __init__(self, head_dim: int, rotary_dim: int | None = None, base: float = 10000.0, scaling: str | None = None,
                 factor: float = 1.0, trained: int | None = None, interleaved: bool = False, device=None):
        dim = head_dim if rotary_dim is None else rotary_dim
        if dim > head_dim:
            raise ValueError(f"rotary_dim {dim} of heads of {head_dim}")
        self.freqs, self.magnitude = ops.rotary_frequencies(dim, base, scaling, factor, trained, device)
        self.interleaved = interleaved

    def __call__(self, x, positions, parents=None) -> torch.Tensor:
        """x [B, T, heads, head_dim] turned to its positions, see ops.rotary."""
        return ops.rotary(x, positions, self.freqs, parents, self.interleaved, self.magnitude)


def decode(blocks: list[DecoderBlock], x: torch.Tensor, cache: PagedCache, parents=None, rotary: Rotary | None = None):
    """The blocks on new tokens x [slots, T, d_model] of every slot, T <= 128, after its cached
    positions: (output [slots, T, d_model], k, v [layers, slots, T, heads, head_dim]). The
    tokens are a tree (parents, see ops.attention_tree) or, without it, follow one another.
    Nothing is kept: append k and v, whole or the accepted path of them. With `rotary` q and k
    are turned to their positions first; the k that comes back is turned."""
    ks, vs = [], []

    def attend(layer, qkv):  # [slots, T, 3, heads, head_dim]
        q, k, v = qkv.unbind(2)
        if rotary is not None:
            q, k = rotary(qkv[:, :, :2].flatten(2, 3), cache.lens, parents).chunk(2, 2)
        ks.append(k)
        vs.append(v)
        return cache.attention(layer, q, k, v, parents)

    return _through(blocks, x, attend), torch.stack(ks), torch.stack(vs)


def extend(blocks: list[DecoderBlock], x: torch.Tensor, cache: PagedCache, rotary: Rotary, count=None) -> torch.Tensor:
    """The blocks on the next tokens x [slots, T, d_model] of every slot, which are kept: prompts, chunk
    by chunk of 128, or one token each. Output [slots, T, d_model]. Pages have to be reserved. count
    [slots]: a slot's number of tokens, those after it are padding, whose output means nothing."""
    T, out = x.shape[1], []
    left = None if count is None else count.clamp(0, T)
    for at in range(0, T, 128):
        part = x[:, at:at + 128]
        n = part.shape[1]
        now = None if left is None else (left - at).clamp(0, n)

        def attend(layer, qkv):
            q, k, v = qkv.unbind(2)
            q, k = cache.write(layer, q, k, v, rotary, now)
            return cache.attention(layer, q, k, v)

        out.append(_through(blocks, part, attend))
        cache._grow(cache.lens + (n if now is None else now))
    if not out:  # no token: nothing is kept
        return x.new_empty(x.shape)
    return torch.cat(out, 1) if len(out) != 1 else out[0]


def _through(blocks: list[DecoderBlock], x: torch.Tensor, attend) -> torch.Tensor:
    """x [slots, T, d_model] through the blocks; attend(layer, qkv) is their attention."""
    B, T, d = x.shape
    for layer, block in enumerate(blocks):
        cfg = block.cfg
        w = device_weights(block, x.dtype, x.device)
        x2 = x.reshape(B * T, d)
        h = ops.rmsnorm(x2, w["norm1"], cfg.eps)
        a = attend(layer, ops.matmul(h, w["wqkv"]).view(B, T, 3, cfg.n_heads, cfg.head_dim))
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
    return x


def _logits(x: torch.Tensor, head: torch.Tensor) -> torch.Tensor:
    x2 = x.reshape(-1, x.shape[-1])
    return torch.ops.nkilab.matmul_f32out(x2, head) if x.dtype == torch.bfloat16 else ops.matmul(x2, head)


def probabilities(x: torch.Tensor, head: torch.Tensor) -> torch.Tensor:
    """softmax(x @ head) in fp32: x [..., d], head [d, V]; V a multiple of 8 for bf16."""
    return ops.softmax(_logits(x, head)).view(*x.shape[:-1], head.shape[1])


def next_token(x: torch.Tensor, head: torch.Tensor, uniforms: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, prob) [slots] drawn from x @ head, x [slots, d], head [d, V]; see ops.sample."""
    return ops.sample(_logits(x, head), uniforms, temperature, top_k, top_p, min_p)


def step(blocks: list[DecoderBlock], embedding: torch.Tensor, head: torch.Tensor, cache: PagedCache, last: torch.Tensor,
         uniforms: torch.Tensor, rotary: Rotary, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token of every slot: `last` [slots], its latest token (not in the cache yet, for which a
    page has to be reserved), goes through the blocks and is kept, and the next one is drawn with the uniform
    numbers [slots]. Returns (token, prob) as ops.sample does. A slot without pages stays empty; one that has ended and
    still has its pages goes on growing: free it, or extend with a count of 0 for it."""
    x = embedding[last.clamp(0, embedding.shape[0] - 1).long()][:, None]
    return next_token(extend(blocks, x, cache, rotary)[:, 0], head, uniforms, temperature, top_k, top_p, min_p)


def speculative_step(blocks: list[DecoderBlock], embedding: torch.Tensor, head: torch.Tensor, cache: PagedCache,
                     last: torch.Tensor, drafts: torch.Tensor, uniforms: torch.Tensor, parents=None, draft_probs=None,
                     rotary: Rotary | None = None):
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
    y, k, v = decode(blocks, embedding[tokens.long()], cache, tree, rotary)
    path, count, token = ops.verify_drafts(probabilities(y, head), drafts, uniforms, parents, draft_probs)
    rows = torch.cat([torch.zeros_like(path[:, :1]), torch.where(path < 0, path, path + 1)], 1)
    cache.append(k, v, rows, count + 1)
    return path, count, token
