"""Host-side ops: the drop-in boundary of the reference's ``nkilab.ops``.

Same names, signatures, argument meaning and error behaviour as the reference
(nkilab/ops.py:1-91 in Nags-gk/nki-kernel-lab): every op takes NumPy arrays (float32
or ml_dtypes.bfloat16) and returns a new NumPy array of the input's dtype, accepts
any shape, and pads / crops internally. Where the reference runs an NKI kernel on
the CPU simulator, these run the B200 CUDA kernels of libnkilab_b200.so through the
``torch.ops.nkilab`` custom ops. They also accept torch tensors: a CUDA tensor stays
on the device (no copies), a CPU tensor (pinned or not) is copied in and the result
copied back to the CPU.

There is no CPU fallback: on a machine without a GPU every op raises.
"""
from __future__ import annotations

import math
import re

import torch

from . import _native
from . import _torch_ops  # noqa: F401  (registers torch.ops.nkilab.*)
from ._host import dtype_of as _dtype_of
from ._host import like_input as _like_input
from ._host import to_device as _to_device
from .kernels import attention as _attn

__all__ = ["choose_blocks", "matmul", "softmax", "rmsnorm", "swiglu", "attention", "ATTENTION_VARIANTS",
           "rope", "attention_tree", "cache_append", "cache_reserve", "cache_fork", "cache_free", "cache_compact",
           "verify_drafts", "rotary_frequencies", "rotary", "rotary_append", "sample"]


# --------------------------------------------------------------------------- matmul

def choose_blocks(m_tiles: int, n_tiles: int) -> tuple[int, int]:
    """Largest BM x BN output block (BM in {1,2,4}, BN in {1,2,4,8}, BM*BN <= 8) dividing
    the (m_tiles, n_tiles) grid; among equal areas the wider block wins.

    Same rule as nkilab/ops.py:27-35 (8 PSUM banks of [128, 512] fp32 per partition on
    Trainium2). The B200 GEMM does not need it -- its output tile lives in TMEM and is
    chosen by the kernel -- but kernels.matmul.matmul_blocked validates block
    arguments against the same budget.
    """
    cands = [(bm, bn) for bm in (1, 2, 4) for bn in (1, 2, 4, 8)
             if bm * bn <= 8 and m_tiles % bm == 0 and n_tiles % bn == 0]
    return max(cands, key=lambda c: (c[0] * c[1], c[1]))


def matmul(a, b, variant: str = "blocked"):
    """C = A @ B for any shapes, fp32 accumulation, output in A's dtype (ops.py:38-52).

    variant "blocked" (default) runs the TMA + tcgen05 GEMM (bf16) or the exact fp32
    CUDA-core GEMM (float32); "naive" runs the no-reuse kernel.
    """
    M, K = a.shape
    K2, N = b.shape
    assert K == K2, (a.shape, b.shape)
    if _dtype_of(a) != _dtype_of(b):
        raise TypeError(f"matmul operands differ in dtype: {_dtype_of(a)} vs {_dtype_of(b)}")
    ad = _to_device(a)
    bd = _to_device(b, ad.device)
    naive = variant == "naive"
    if ad.dtype == torch.bfloat16 and not naive and (K % 8 or N % 8):
        # TMA rows must be 16-byte multiples: zero-pad K and N to multiples of 8 (the
        # padded products are zeros), then crop, as the reference pads to its tiles.
        Kp, Np = -(-K // 8) * 8, -(-N // 8) * 8
        ad = torch.nn.functional.pad(ad, (0, Kp - K))
        bd = torch.nn.functional.pad(bd, (0, Np - N, 0, Kp - K))
        c = torch.ops.nkilab.matmul(ad, bd, False)[:, :N].contiguous()
    else:
        c = torch.ops.nkilab.matmul(ad, bd, naive)
    return _like_input(c, a)


# --------------------------------------------------------------------------- row kernels

def softmax(x, fused: bool = True):
    """Row softmax over the last dim (ops.py:55-57): fused single pass, or the 3-pass
    unfused kernel sequence when fused=False."""
    xd = _to_device(x)
    return _like_input(torch.ops.nkilab.softmax(xd, bool(fused)), x)


def rmsnorm(x, weight, eps: float = 1e-6):
    """y = x * rsqrt(mean(x^2) + eps) * weight over the last dim (ops.py:60-61)."""
    xd = _to_device(x)
    wd = _to_device(weight, xd.device)
    if wd.dtype != xd.dtype:
        wd = wd.to(xd.dtype)
    return _like_input(torch.ops.nkilab.rmsnorm(xd, wd, float(eps)), x)


def swiglu(gate, up):
    """y = silu(gate) * up elementwise (ops.py:64-65)."""
    gd = _to_device(gate)
    ud = _to_device(up, gd.device)
    return _like_input(torch.ops.nkilab.swiglu(gd, ud), gate)


# --------------------------------------------------------------------------- attention

ATTENTION_VARIANTS = {
    "naive": _attn.attention_naive,
    "flash": _attn.flash_attention,
    "flash_kv_resident": _attn.flash_attention_kv_resident,
    "flash_balanced": _attn.flash_attention_balanced,
    "flash_pipelined": _attn.flash_attention_pipelined,
}


def attention(q, k, v, variant: str = "flash_pipelined"):
    """Causal attention, q, k, v: [H, S, d], scale 1/sqrt(d) (ops.py:77-91).

    Any S: the kernels handle a partial last tile directly, so there is no host
    padding of the sequence. bf16 head dims other than 64/128 are zero-padded to the
    next of those (padding q/k columns adds zeros to every score; padded v columns
    are cropped). Every "flash*" variant runs the same tcgen05 flash kernel (the
    reference's variants share numerics, tests/test_attention.py:67-70);
    "naive" materialises the scores and probabilities.

    Extension beyond the reference: k and v may carry fewer heads than q (grouped-query
    or multi-query attention); query head h then uses key/value head h // (H // Hkv).
    """
    if variant not in ATTENTION_VARIANTS:
        raise KeyError(variant)
    H, S, d = q.shape
    assert d <= 128, f"head_dim {d} > 128"
    qd = _to_device(q)
    kd = _to_device(k, qd.device)
    vd = _to_device(v, qd.device)
    scale = 1.0 / math.sqrt(d)
    naive = variant == "naive"
    dp = d
    if qd.dtype == torch.bfloat16 and not naive and d not in (64, 128):
        dp = 64 if d < 64 else 128
        pad = (0, dp - d)
        qd, kd, vd = (torch.nn.functional.pad(t, pad) for t in (qd, kd, vd))
    o = torch.ops.nkilab.attention(qd, kd, vd, scale, naive)
    if dp != d:
        o = o[..., :d].contiguous()
    return _like_input(o, q)


def rope(x, base: float = 10000.0, pos_offset: int = 0):
    """Rotary position embedding, rotate-half convention, of x: [H, S, d] (extension
    beyond the reference, which lists rotary embeddings as not done, README.md:89).
    Position of row s is s + pos_offset; theta_i = base^(-2i/d). NumPy or torch in,
    same kind out."""
    xd = _to_device(x).contiguous()
    o = torch.ops.nkilab.rope(xd, float(base), int(pos_offset))
    return _like_input(o, x)


# --------------------------------------------------------------------------- decoding (extension)
# Operations of a decoding loop on a paged key/value cache. The cache lives on the GPU, so
# these take CUDA tensors only. Shapes: caches [pages, kv heads, page size, head_dim], with a
# leading [layers] for the page operations where there are several; tables [B, M] int32, the
# pages of each slot in order (-1: none); lens [B] int32, cached positions of each slot; refs
# [pages] int32, how many table entries name each page. Nothing here reads them on the host
# or waits for the GPU. nkilab.serving.PagedCache keeps them together.

def _decode(name: str):
    """torch.ops.nkilab.<name>, with a refusal of the C ABI raised as NklError."""
    op = getattr(torch.ops.nkilab, name).default

    def call(*args):
        try:
            return op(*args)
        except RuntimeError as e:
            m = re.match(r"(nkl_\w+) failed \((\d+)\): ([^\n]*)", str(e))
            if type(e) is not RuntimeError or m is None:
                raise
            raise _native.NklError(m[1], int(m[2]), m[3]) from None

    return call


_attention_tree, _cache_append, _cache_reserve, _cache_fork, _cache_free, _cache_compact, _verify_drafts = map(
    _decode, ("attention_tree", "cache_append", "cache_reserve", "cache_fork", "cache_free", "cache_compact",
              "verify_drafts"))
_attention_tree_8bit, _cache_append_8bit, _cache_fork_8bit, _cache_compact_8bit, _rotary, _rotary_append, _sample = map(
    _decode, ("attention_tree_8bit", "cache_append_8bit", "cache_fork_8bit", "cache_compact_8bit", "rotary", "rotary_append",
              "sample"))


def attention_tree(q, k, v, k_cache, v_cache, tables, lens, parents=None, scale=None, k_scales=None, v_scales=None):
    """Attention of T drafted tokens per sequence over its cached positions and, as a tree,
    over each other. q: [B, T, H, d]; k, v: [B, T, Hkv, d], the drafted tokens' own, not yet
    in the cache (views of a fused projection are read as they lie); returns [B, T, H, d].

    parents [B, T] int32: each token's parent among the earlier ones, -1 for a child of the
    last cached position, -2 for an absent token (its output is zero, none sees it). None:
    each token follows the one before it, so T = 1 is plain decoding and T > 1 a chunk of a
    prompt. At most 128 tokens; scale defaults to 1/sqrt(d). d: a multiple of 8 up to 128
    (64 and 128 in bf16, with pages of a multiple of 8 positions, run on tcgen05). There is
    no backward pass: one through it raises, as does a forward derivative.

    With k_scales and v_scales the caches are in 8 bits, as cache_append writes them (d a multiple
    of 16); q, k and v are bf16 or fp32 all the same.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if k_scales is not None or v_scales is not None:
        if k_scales is None or v_scales is None:
            raise ValueError("scales: need both or none")
        return _attention_tree_8bit(q, k, v, k_cache, v_cache, k_scales, v_scales, tables, lens, parents, float(scale))
    return _attention_tree(q, k, v, k_cache, v_cache, tables, lens, parents, float(scale))


def cache_append(k, v, k_cache, v_cache, tables, lens, path=None, count=None, k_scales=None, v_scales=None):
    """Writes rows of k and v [(layers,) B, T, Hkv, d] to the pages at positions lens[b]
    onward and returns the new lengths: row path[b, j] for j < count[b] (the accepted path
    of drafted tokens), or all T rows in order. The pages come from cache_reserve; rows
    without a page are dropped, but counted in the lengths (PagedCache.append bounds them).

    With k_scales and v_scales [(layers,) pages, Hkv, blocks of a page] float8_e8m0fnu the caches are
    float8_e4m3fn (d a multiple of 16 up to 128) and a value is number * scale. Each block of
    page / blocks positions has the smallest power of two, from 2^-100 on, with which its largest
    magnitude is at most 448 of it; rows of a block that grows past its power are rounded again. An
    infinity or NaN makes its block NaN."""
    if k_cache.dim() == 4:  # one layer
        k, v, k_cache, v_cache = (t.unsqueeze(0) for t in (k, v, k_cache, v_cache))
        k_scales, v_scales = (t if t is None else t.unsqueeze(0) for t in (k_scales, v_scales))
    if k_scales is None and v_scales is None:
        return _cache_append(k, v, k_cache, v_cache, tables, lens, path, count)
    if k_scales is None or v_scales is None:
        raise ValueError("scales: need both or none")
    return _cache_append_8bit(k, v, k_cache, v_cache, k_scales, v_scales, tables, lens, path, count)


ROTARY_SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, trained=None, device=None):
    """(freqs, magnitude) for `rotary`: freqs [rotary_dim / 2] float64, radians to a position, base^(-2i /
    rotary_dim), stretched by `factor` for contexts longer than the `trained` one:

    "linear"  every frequency / factor (positions interpolated)
    "ntk"     base * factor^(r / (r - 2)), which divides the lowest frequency by factor
    "yarn"    frequencies that turn less than once in `trained` positions / factor, those that turn
              over 32 times as they are, mixed linearly between, by the number of turns; magnitude
              0.1 ln(factor) + 1 (Peng et al., YaRN, 2023). Implementations that mix linearly by the pair's
              index have other frequencies in between: a model trained with those needs its own `freqs`
    """
    r = int(rotary_dim)
    if r < 2 or r % 2:
        raise ValueError(f"rotary_dim {rotary_dim}: must be even and positive")
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"scaling {scaling!r}: one of {ROTARY_SCALINGS}")
    if not (base > 1 and factor >= 1):
        raise ValueError(f"base {base}, factor {factor}: need base > 1 and factor >= 1")
    if scaling == "yarn" and not trained:
        raise ValueError("yarn: needs the number of trained positions")
    if scaling == "ntk":
        if r < 4:
            raise ValueError("ntk: needs a rotary_dim of 4 or more")
        base = base * factor ** (r / (r - 2))
    f = float(base) ** (-2 * torch.arange(r // 2, dtype=torch.float64) / r)
    magnitude = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        stay = ((trained * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * (stay + (1 - stay) / factor)
        magnitude = 0.1 * math.log(factor) + 1
    return f.to(torch.device("cuda", torch.cuda.current_device()) if device is None else device), magnitude


def rotary(x, positions, freqs, parents=None, interleaved=False, magnitude=1.0):
    """Rotary positions of x [B, T, heads, d] (queries and keys of a fused projection together, as
    they lie): the first 2 len(freqs) entries of a head are pairs (i, i + len(freqs)), or (2i, 2i + 1) if
    `interleaved`, turned by position * freqs[i] and times magnitude; the rest stays. Both sizes are
    multiples of 8, d up to 256.

    positions int32: [B, T], or [B], where token j is at positions[b] + j, or, in a tree (parents
    [B, T] as in attention_tree), as far behind as it is deep. Angles are reduced in 64 bits. x may
    need a gradient, which turns the other way, or have a forward derivative, which turns along.
    """
    return _rotary(x, positions, freqs, parents, bool(interleaved), float(magnitude), False)


def rotary_append(q, k, v, k_cache, v_cache, tables, lens, freqs, count=None, interleaved=False, magnitude=1.0,
                  k_scales=None, v_scales=None):
    """q [B, T, H, d] and k [B, T, Hkv, d] turned as by `rotary` at positions lens[b] + j, and the
    turned k and v written to those positions of one layer's cache (in 8 bits with scales, see
    cache_append; rounded once there). Returns (q, k). Rows from count[b] on stay out of
    the cache, as do rows without a page; lens stays as it is, for a step's layers share it. There
    is no backward pass: one through it raises, as does a forward derivative.
    """
    return _rotary_append(q, k, v, k_cache, v_cache, k_scales, v_scales, tables, lens, freqs, count, bool(interleaved),
                          float(magnitude))


def cache_reserve(tables, lens, refs, extra, page_size):
    """Pages for extra[b] more positions of each slot, lowest free index first. Returns
    (tables, refs, missing): with too few free pages, or too narrow tables, missing [1] is
    how many lack and nothing is given out."""
    return _cache_reserve(tables, lens, refs, extra, int(page_size))


def _check_8bits(k_cache, v_cache, k_scales, v_scales):
    """Caches in 8 bits have both scales, others none."""
    if (k_scales is None) != (v_scales is None):
        raise ValueError("scales: need both or none")
    for c in (k_cache, v_cache):
        if (c.dtype == torch.float8_e4m3fn) != (k_scales is not None):
            raise TypeError(f"a {c.dtype} cache {'without' if k_scales is None else 'with'} scales")


def cache_fork(k_cache, v_cache, tables, lens, refs, src, dst, k_scales=None, v_scales=None):
    """Slot dst[f] becomes a copy of slot src[f]: full pages are shared, the last, partly
    filled one is copied to a free page. Returns (tables, lens, refs, missing); with
    missing [1] > 0 (too few free pages) nothing is forked. A cache in 8 bits needs its scales, which go along."""
    if k_scales is not None or v_scales is not None or k_cache.dtype == torch.float8_e4m3fn:
        _check_8bits(k_cache, v_cache, k_scales, v_scales)
        if k_cache.dim() == 4:  # one layer
            k_cache, v_cache, k_scales, v_scales = (t.unsqueeze(0) for t in (k_cache, v_cache, k_scales, v_scales))
        return _cache_fork_8bit(k_cache, v_cache, k_scales, v_scales, tables, lens, refs, src, dst)
    if k_cache.dim() == 4:  # one layer
        k_cache, v_cache = k_cache.unsqueeze(0), v_cache.unsqueeze(0)
    return _cache_fork(k_cache, v_cache, tables, lens, refs, src, dst)


def cache_free(tables, lens, refs, slots):
    """Gives back the pages of the slots listed. Returns (tables, lens, refs)."""
    return _cache_free(tables, lens, refs, slots)


def cache_compact(k_cache, v_cache, tables, refs, k_scales=None, v_scales=None):
    """Moves the pages in use to the lowest indices. Returns (tables, refs). A cache in 8 bits needs
    its scales, which go along."""
    if k_scales is not None or v_scales is not None or k_cache.dtype == torch.float8_e4m3fn:
        _check_8bits(k_cache, v_cache, k_scales, v_scales)
        if k_cache.dim() == 4:  # one layer
            k_cache, v_cache, k_scales, v_scales = (t.unsqueeze(0) for t in (k_cache, v_cache, k_scales, v_scales))
        return _cache_compact_8bit(k_cache, v_cache, k_scales, v_scales, tables, refs)
    if k_cache.dim() == 4:  # one layer
        k_cache, v_cache = k_cache.unsqueeze(0), v_cache.unsqueeze(0)
    return _cache_compact(k_cache, v_cache, tables, refs)


def verify_drafts(probs, tokens, uniforms, parents=None, draft_probs=None):
    """Accepts drafted tokens against the target's probabilities and draws the next token, so
    that the tokens are distributed as the target's. probs [B, T + 1, V]: row 0 after the last
    cached token, row i + 1 after drafted token i; tokens [B, T] int32; uniforms [B, T + 1]
    float32 in [0, 1). A chain with draft_probs [B, T, V] (what each token was drawn from), or
    a tree with parents [B, T] (None: a chain) and no draft_probs. Absent tokens and their
    children are never accepted.

    Returns (path [B, T], the accepted tokens' indices and then -1; count [B]; token [B]).
    Sums are whole numbers of 2^-31, so equal inputs give equal tokens on every launch.
    """
    return _verify_drafts(probs, tokens, uniforms, parents, draft_probs)


def sample(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The next token of each row of logits [B, V] from the uniform numbers [B] (float32 in [0, 1)).

    Weights are exp((x - max) / temperature); tokens in order of their logits, of equal ones the
    lowest index first, are kept while they are among the first top_k, needed for the share top_p of
    the top_k's weights, and weigh at least min_p of the first one; the first one always is. temperature
    0 takes the first one; top_k 0, top_p 1 and min_p 0 keep all. Each is a number, or one for each row: a
    tensor [B] on the GPU (top_k int32, the others float32), where NaN is off. Minus infinity and NaN are never
    drawn. Returns (token [B] int32, -1 if there is none; prob [B] float32, its share of what was kept).
    Weights are whole multiples of 2^-31 (the formula's, rounded down, to within one), so equal inputs give equal tokens on
    every launch. V up to 360448. No derivative passes through it: one that is asked for raises.
    """
    numbers, rows = [], []
    for name, x, low, high in (("temperature", temperature, 0, math.inf), ("top_k", top_k, 0, 2 ** 31), ("top_p", top_p, 0, 1),
                               ("min_p", min_p, 0, 1)):
        each = isinstance(x, torch.Tensor)
        if not each and not low <= x <= high:
            raise ValueError(f"{name} {x}: must be between {low} and {high}")
        rows.append(x if each else None)
        numbers.append(0 if each else x)
    return _sample(logits, uniforms, *rows, float(numbers[0]), int(numbers[1]), float(numbers[2]), float(numbers[3]))
