"""Generating with a key/value cache in 8 bits.

``GPTModel.generate`` (model.py:316-355) runs the whole sequence through every layer again for each new token. With a cache
a layer appends the new tokens' keys and values (``cache_append``) and attends from the new tokens alone (``cache_attention``),
with the mask of ``flash_attention``: the 4-section rule when the cache holds metadata, else causal. Where memory is short,
``cache_attention`` adds up the weight that every cached token receives, and ``cache_evict`` keeps the tokens that received most of it.

Format. Pages of 64 tokens: ``k`` and ``v`` float8_e4m3fn (pages, heads, 64, head_dim), ``k_scale`` and ``v_scale`` float32 (pages, heads).
A stored number stands for its value times the scale of its page and head: 2**e with -32 <= e <= 31, the smallest e that lets the block's
largest finite magnitude be at most 448 * 2**e. Larger numbers saturate; infinities and NaN are stored as NaN. A block that receives tokens
later keeps its scale or gets a larger one, and what it holds is rounded again: exactly, but for numbers that become subnormal.
``desc`` (optional) holds the mask descriptor of every token: int32, bit 0 prefix, 1 context, 2 in a span, 3 [MASKQ], 4 same-span rule armed,
5 to 7 the classes of keys that the token sees wherever they are, from 8 the span id.

Sequences. ``page_table`` int32 (batch, blocks) names the pages of every sequence in order, ``lens`` int32 (batch,) counts its tokens; both
stay on the device, so that a step can be captured into a CUDA graph. Pages are the caller's to hand out. What the table holds behind a
sequence's last block is not read. Sequences may share pages as long as none of them appends to one. A length that the table has no
pages for, or a page that does not exist, is no fault: the excess is left out (``cache_append`` writes nothing to a sequence whose length or number of new tokens cannot be), and the next call with the cache raises ``ValueError``
(with ``KD_CHECK_STATUS=1`` the same one, which then waits for the device).

There is no backward: inputs that require gradients are refused unless gradients are off.
"""
from __future__ import annotations

import torch

from . import _host

_ext = _host.load()

__all__ = ["KVCache", "cache_append", "cache_attention", "cache_evict", "cache_read"]

#: tokens of a page
PAGE = 64


class KVCache:
    """A pool of pages: the five tensors of the format, which stay the caller's."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "desc", "_core")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, desc: torch.Tensor | None = None):
        self._core = _ext.KVCache(k, v, k_scale, v_scale, desc)
        self.k, self.v, self.k_scale, self.v_scale, self.desc = k, v, k_scale, v_scale, desc

    @classmethod
    def empty(cls, pages: int, heads: int, head_dim: int, device="cuda", metadata: bool = False) -> "KVCache":
        """A new pool; ``metadata``: with room for the mask descriptors."""
        k, v = (torch.zeros((pages, heads, PAGE, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
        scales = torch.ones((2, pages, heads), dtype=torch.float32, device=device)
        desc = torch.zeros((pages, heads, PAGE), dtype=torch.int32, device=device) if metadata else None
        return cls(k, v, scales[0].clone(), scales[1].clone(), desc)


def cache_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor,
                 new_lens: torch.Tensor | None = None, in_span: torch.Tensor | None = None, span_id: torch.Tensor | None = None,
                 is_prefix: torch.Tensor | None = None) -> None:
    """Puts new keys and values behind the ``lens[b]`` tokens of every sequence. ``lens`` is not changed: the caller adds.

    k, v: (batch, cache heads, time, head_dim) float16, bfloat16 or float32, any strides. new_lens: int32 (batch,), how many of
    the ``time`` tokens a sequence really has (None: all); the rest, and every slot behind them in a block that held tokens, stays as
    it was. in_span / is_prefix bool and span_id int64 (batch, time): the new tokens' metadata as for ``flash_attention`` (a missing one
    is all zeros; a span_id beyond 24 signed bits is reported as a bad length is), for a cache with ``desc``."""
    _ext.cache_append(cache._core, k, v, page_table, lens, new_lens, in_span, span_id, is_prefix)


def cache_attention(q: torch.Tensor, cache: KVCache, page_table: torch.Tensor, lens: torch.Tensor, q_lens: torch.Tensor | None = None,
                    sm_scale: float | None = None, causal: bool = True, return_lse: bool = False, weights: torch.Tensor | None = None,
                    out_layout: str = "contiguous"):
    """Attention of every sequence's newest tokens over all its cached ones, their own keys and values among them.

    q: (batch, heads, time, head_dim) float16 or bfloat16, any strides; heads a multiple of the cache's (query head h reads key
    head h // (heads // cache heads)). Query i of sequence b is its token ``lens[b] - q_lens[b] + i``; q_lens int32 (batch,), None:
    ``time`` for all. The mask is the 4-section rule of ``flash_attention`` when the cache holds metadata (``causal`` is not part of it then),
    otherwise ``j <= i`` (causal) or every cached token. Rows at or beyond ``q_lens``, and rows that see nothing, get O = 0 and LSE = -inf.

    weights: float32 (batch, cache heads, tokens), to which the softmax weight is added that each cached token receives from all queries of
    its head; tokens beyond its last dimension are left out. sm_scale: head_dim ** -0.5 by default. out_layout: "contiguous", or "input" for O in
    the memory layout of q.

    A weight enters the product with v with 11 bits, and with an error of no more than 2**-28 of the row's largest weight (2**-25 in rows with scores
    beyond 2**16, in powers of two), or, where the value scales of pages are more than 2**4 apart, 2**-20 of its page's largest.

    Returns O in the type of q, or (O, LSE) with ``return_lse`` (float32 (batch, heads, time), base 2)."""
    if out_layout not in ("contiguous", "input"):
        raise ValueError("out_layout must be 'contiguous' or 'input'")
    o, lse = _ext.cache_attention(cache._core, q, page_table, lens, q_lens, sm_scale, causal, return_lse, weights, out_layout == "input")
    return (o, lse) if return_lse else o


def cache_evict(cache: KVCache, page_table: torch.Tensor, lens: torch.Tensor, weights: torch.Tensor, out_table: torch.Tensor, keep: int,
                recent: int = 0, first: int = 0):
    """Keeps up to ``keep`` tokens of every sequence and head: its first ``first``, its last ``recent``, and of the others those of the
    largest accumulated weight (of equal ones the earlier; NaN counts as largest). A sequence that has no more keeps them all.

    The kept tokens go in their order to the pages that out_table (batch, at least ceil(keep / 64) blocks) names, as if they had been appended there;
    these pages must not be among those of page_table. The old pages are left as they are, for the caller to hand out again. The heads of a
    sequence keep different tokens, which ``cache_attention`` does not notice: a later query is behind all of them.

    weights: float32 (batch, cache heads, tokens) as ``cache_attention`` fills it; a token beyond it weighs nothing.
    Returns (index int32 (batch, heads, keep), lens int32 (batch,), weights float32 (batch, heads, keep)): the kept tokens' places,
    ascending, -1 behind the last; the new lengths; the kept tokens' weights, 0 behind the last."""
    return _ext.cache_evict(cache._core, page_table, lens, weights, out_table, keep, recent, first)


def cache_read(cache: KVCache, page_table: torch.Tensor, lens: torch.Tensor, count: int, start: torch.Tensor | None = None,
               dtype: torch.dtype = torch.bfloat16):
    """(k, v), each (batch, cache heads, count, head_dim): the values of the cached tokens start[b] .. start[b] + count - 1 (start int32
    (batch,), None: 0), zeros where a sequence has none. bfloat16 and float32 hold every cached number exactly; float16 those in its range."""
    return _ext.cache_read(cache._core, page_table, lens, count, start, dtype)
