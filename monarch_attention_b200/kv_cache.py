"""A paged cache of keys and values in 8 bits, and softmax attention of new tokens over it.

The other half of an encoder with :class:`MonarchAttention`: its decoder answers a token at a time, and each token's attention
reads the keys and values of all before it (or of the encoder's output).  Both live here in pages of a pool, so that sequences of
different lengths share memory, in e4m3 with a power-of-two scale for each block of 16 tokens of a head.  The kernels are
``ma_b200_cache_append`` and ``ma_b200_cache_attend`` of the library; nothing here runs on the CPU.

Which tokens a call is about is said the same way everywhere: ``page_table`` (E, P) int32, the page of each run of ``page_size`` tokens of a
sequence; ``lengths`` (E) int32, the tokens of each sequence, those of the call among them; ``counts`` (E) int32 or None, how many of
the call's N tokens are a sequence's own (the rest is padding behind them).  Token n of the call stands at position
``lengths[e] - counts[e] + n``.  The three are read on the GPU, so that nothing waits for the host and calls can be captured in a
graph.  A length that the table has no room for, a count above N or a page outside the cache is not followed: what
it concerns is left out or undefined, and a later call on the device raises ``RuntimeError``.  A count above the length is one of these when
appending; in the attention, rows in front of a sequence's first token see no key and are zero.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn as nn

from .rotary import RotaryPositions

Tensor = torch.Tensor

BLOCK = 16  # tokens that share a scale
_NO_ROTARY = (None, 0, 0, 1.0)


class PagedKV(NamedTuple):
    """The pool: ``k``, ``v`` (pages, heads, page size, width) float8_e4m3fn and ``k_scale``, ``v_scale`` (pages, heads, page size / 16) float32.

    The 16 tokens of a block of a head stand for ``code * scale`` (scales are not negative, and zero or from 2^-40 to 2^60).  The width is 64 or 128, the page size a power of two from 16 on; strides
    are free as long as rows start on 16-byte boundaries (a pool of (pages, page size, heads, width) is passed as a permuted view).
    """

    k: Tensor
    v: Tensor
    k_scale: Tensor
    v_scale: Tensor

    @classmethod
    def allocate(cls, pages: int, heads: int, width: int, page_size: int = 64, device="cuda") -> "PagedKV":
        """An empty pool."""
        if width not in (64, 128):
            raise ValueError(f"width must be 64 or 128, got {width}")
        if page_size < BLOCK or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from {BLOCK} on, got {page_size}")
        if pages <= 0 or heads <= 0:
            raise ValueError("pages and heads must be positive")
        codes = [torch.zeros(pages, heads, page_size, width, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
        scales = [torch.zeros(pages, heads, page_size // BLOCK, dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)


_append = _attend = None


def _load() -> None:
    global _append, _attend
    from .monarch_attention import native_module
    native = native_module()
    _append, _attend = native.append, native.attend


def append_kv_b200(cache: PagedKV, key: Tensor, value: Tensor, page_table: Tensor, lengths: Tensor, counts: Tensor | None = None, *,
                   query: Tensor | None = None, rotary: RotaryPositions | None = None, parents: Tensor | None = None) -> Tensor | None:
    """Writes ``key`` and ``value`` (E, heads, N, width; bfloat16 or float16) into the cache at the call's positions.

    With ``rotary`` (``dim`` a multiple of 16) keys are rotated at their positions on the way, and so is ``query`` (E, H, N, width), whose
    rotated copy is returned, with rows of padding as zeros.  A block's scale is the smallest power of two from 2^-40 to 2^60 with which 448 holds the
    block's largest magnitude.  It never falls while the block has older tokens; when it rises they are re-expressed, which is exact but for
    values that become subnormal.  Magnitudes above 448 * 2^60 (infinities) are stored as that, NaN as NaN.  The pages that a call writes to
    must stand once in one sequence's row of the table (pages that are only read may be shared), and the pool's pages, heads and tokens must not
    overlap (keys and values may lie in one buffer, with the same strides).  No gradient: inputs that require one are refused.

    ``parents`` (E, N; int32, N up to 512): the tokens are a tree, several continuations of a sequence at once.  Each names its parent, an earlier token of the call, or -1.  A
    token lies in the cache at its place in the call, and is rotated at the position of its depth: ``lengths[e] - counts[e]`` and the number of its ancestors.
    """
    if _append is None:
        _load()
    if rotary is not None and not isinstance(rotary, RotaryPositions):
        raise TypeError("rotary must be a RotaryPositions or None")
    return _append(*cache, key, value, page_table, lengths, counts, query, *(rotary._native if rotary is not None else _NO_ROTARY),
                   parents)


def cached_attention_b200(query: Tensor, cache: PagedKV, page_table: Tensor, lengths: Tensor, counts: Tensor | None = None, *,
                          causal: bool = True, scale: float | None = None, softcap: float = 0.0, window: int = 0,
                          parents: Tensor | None = None, out: Tensor | None = None, token_major_output: bool = False) -> Tensor:
    """Softmax attention of ``query`` (E, H, N, width; bfloat16 or float16) over the cached tokens of its sequences.

    Query head ``h`` reads cache head ``h // (H / heads)``.  ``causal``: a token sees the positions up to its own (the call's tokens have been
    appended before); else all ``lengths`` (an encoder's output).  ``window`` > 0 (causal only): the last ``window`` of those.  Scores are
    multiplied by ``scale`` (None: ``width ** -0.5``) and, with ``softcap`` > 0 (from 1e-20 to 1e30), become ``softcap * tanh(score / softcap)``.  Rows without
    a key, and rows of padding, are zero.  What lies in the cache behind a sequence's end is never looked at, NaN included; a NaN that was appended as a key
    makes NaN of the rows that see it, as a value it reaches all of the call's rows of its sequence and head, masked ones too (zero times NaN).

    ``parents`` (E, N; int32, N up to 512; causal only): the call's tokens are a tree, appended with the same parents.  A token sees what is cached in front of
    the call, its ancestors and itself; a window counts positions, which go by depth.  A parent that is no earlier token of the call counts as -1, none, and a
    later call raises.

    The result has the query's dtype, and with ``token_major_output`` is a view of an (E, N, H, width) buffer; ``out`` (rows on 16-byte
    boundaries) takes it in place: the query itself, or rows beside its own in a common buffer, are fine; rows over one another or over others of the
    query's are refused.  Scores and sums are in 32 bits; a bfloat16 query is read in 16-bit steps of 2^-11 of itself and 2^-25 of its row's
    largest magnitude.  Weights, each times its value's scale, are rounded to 2^-11 of themselves or 2^-32 of their row's largest, whichever is more; what
    is below 2^-25 of a sum so far may be lost from it, as 32 bits have it.  Where scores pass 2^27 and there are 32 rows or fewer to a cache head
    (tokens times query heads of it), scales of values are to be from 2^-14 to 2^15.  The same call gives the same bits; what else is in the batch may
    change the order of a sequence's sums.  No gradient: inputs that require one are refused.
    """
    if _attend is None:
        _load()
    return _attend(query, *cache, page_table, lengths, counts, causal, query.shape[-1] ** -0.5 if scale is None else scale, softcap, window,
                   out, token_major_output, parents)


class CachedAttention(nn.Module):
    """The attention of a decoder layer: new tokens into the cache, then attention over all of it.

    ``forward(query, key, value, cache, page_table, lengths, counts=None, parents=None)`` has query, key and value of one step (a prompt, a piece of
    one, or a token) in the (E, H, N, width) views that :class:`MonarchAttention` takes, key and value with the cache's heads.  With
    ``key`` and ``value`` None nothing is appended and the query is not rotated: attention to an encoder's output that is in the cache already.
    With ``parents`` (``causal`` only) the step's tokens are a tree of drafted ones (:func:`accept_drafts_b200` then keeps those that the model confirms).
    """

    def __init__(self, rotary: RotaryPositions | None = None, causal: bool = True, scale: float | None = None, softcap: float = 0.0,
                 window: int = 0):
        super().__init__()
        if window < 0 or (window and not causal):
            raise ValueError("window must not be negative, and needs causal")
        self.rotary, self.causal, self.scale, self.softcap, self.window = rotary, causal, scale, softcap, window
        # Set to True to get the result as a view of a (batch, tokens, heads, width) buffer, as MonarchAttention has it.
        self.token_major_output = False

    def forward(self, query, key, value, cache, page_table, lengths, counts=None, parents=None):
        if (key is None) != (value is None):
            raise ValueError("key and value must be given together")
        if parents is not None and not self.causal:  # (before the append changes the cache)
            raise ValueError("parents need causal: a tree's tokens see their ancestors")
        if key is not None:
            rotated = append_kv_b200(cache, key, value, page_table, lengths, counts, query=query if self.rotary is not None else None,
                                     rotary=self.rotary, parents=parents)
            query = rotated if self.rotary is not None else query
        return cached_attention_b200(query, cache, page_table, lengths, counts, causal=self.causal, scale=self.scale, softcap=self.softcap,
                                     window=self.window, parents=parents, token_major_output=self.token_major_output)

    def extra_repr(self) -> str:
        return f"rotary={self.rotary}, causal={self.causal}, softcap={self.softcap}, window={self.window}"
