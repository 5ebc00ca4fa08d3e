"""What happens to the sequences of a paged cache between a decoder's steps: drafts are accepted, sequences fork, end, and get pages.

Both operators are about the caches of all layers at once (``caches``: a :class:`PagedKV` or a sequence of them, of one shape and the same strides, none over another),
which share a page table.  Nothing waits for the host, so a step that ends with them can be captured in a graph.  What the tables get wrong is left out, and a later
call on the device raises ``RuntimeError``, as with the append and the attention (``kv_cache.py``).
"""
from __future__ import annotations

from collections.abc import Sequence
from typing import NamedTuple

import torch

from .kv_cache import PagedKV

Tensor = torch.Tensor


class AcceptedDrafts(NamedTuple):
    """``lengths`` (E) int32: tokens of each sequence now; ``path`` (E, N) int32: the call's tokens that stand, in order, -1 behind them; ``answer`` (E): what the model
    answered the last of them with (-1 where none stands)."""

    lengths: Tensor
    path: Tensor
    answer: Tensor


_accept = _fork = None


def _load() -> None:
    global _accept, _fork
    from .monarch_attention import native_module
    native = native_module()
    _accept, _fork = native.accept, native.fork


def accept_drafts_b200(caches: PagedKV | Sequence[PagedKV], page_table: Tensor, lengths: Tensor, counts: Tensor | None, parents: Tensor, drafted: Tensor,
                       answers: Tensor) -> AcceptedDrafts:
    """Which tokens of a tree stand, and the caches closed up over them.

    ``page_table``, ``lengths``, ``counts`` and ``parents`` are those of the step that appended the tree; ``drafted`` (E, N; int32 or int64) its tokens and
    ``answers`` (E, N) what the model answers each with.  A sequence's token 0 stands: it is the model's own last answer.  Another one stands if its parent does and
    it is what the parent was answered with (the first of several).  A choice that is made elsewhere (by rejection sampling, say) is given the same way, as
    answers that name the chosen children.

    The tokens that stand move to the places right behind what was cached before the step, where their depth has put them in the rotation already.  Values stay what they
    are: a block that tokens move into has the smallest scale that holds them, as an append would give it, but where older tokens stay in the block no less than it has, and codes
    move by whole exponents, exact but for values that become subnormal (scales that are no powers of two cost a rounding).  A rejected token may have raised the scale of a block
    that it shared with older ones, and that stays: where it was of far larger magnitude, small values of up to 15 tokens that stand have lost bits, or become zero.  As with the append, pages from the call's first token on must stand once in one sequence's row.  ``lengths`` is not changed; the new ones are returned.  The pages behind the new ends stay with their rows
    (:func:`fork_sequences_b200` gives them back).  A count above N or the length is none.
    """
    if _accept is None:
        _load()
    return AcceptedDrafts(*_accept((caches,) if isinstance(caches, PagedKV) else caches, page_table, lengths, counts, parents, drafted, answers))


def fork_sequences_b200(caches: PagedKV | Sequence[PagedKV], page_uses: Tensor, page_table: Tensor, lengths: Tensor, source: Tensor | None = None,
                        room: Tensor | int = 0) -> None:
    """Sequences go on from others, end, and get room; ``page_uses``, ``page_table`` and ``lengths`` are changed in place.

    ``page_uses`` (pages) int32: how many rows of the table hold each page (zeros at the start; a pool may have several tables, which share the counts).  A row of
    ``page_table`` (E, P; int32) holds the pages in front of its first negative entry (-1 throughout at the start).  ``lengths`` (E) int32: tokens of each sequence.

    Row ``e`` takes what row ``source[e]`` (int32; None: each its own) held before the call, all rows at once, so that rows can be exchanged; -1: it ends and
    holds nothing.  Full pages are shared.  The pages behind them, the first of which may hold some tokens, stay with one row, ``source[e]`` itself if it goes on from itself,
    else the first that goes on from it; each other row gets a copy of those tokens, in all layers, and so does every row whose page another row holds too.  After the
    call no page that an append would write to is held twice.

    ``room`` (E; int32, or one number for all): each row ends with pages for ``lengths + room`` tokens, and gives back what it held beyond.  A new sequence is a row of length 0 (its source
    -1, say) with room for its prompt.  New pages are the lowest free ones, in the order of rows; a pool without enough of them is reported, and the rows that got
    none end where their pages do.  A source that is no row counts as the row itself, and is reported.
    """
    if _fork is None:
        _load()
    _fork((caches,) if isinstance(caches, PagedKV) else caches, page_uses, page_table, lengths, source, room)
