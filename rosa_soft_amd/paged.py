"""Full attention for serving, over a paged cache that the slots of a server share.

The mixers' updates keep a state, or the last tokens, of every slot.  Attention over all that a slot
holds needs memory by its length, which differs from slot to slot and grows with every token: keys and
values lie on pages of one pool, and a table for each slot says which.

* ``page_tables_update`` hands pages to the slots' new tokens and says on which row each lies,
  ``page_tables_release`` takes them back from ended requests and rejected tokens;
* ``paged_attention_update`` puts new tokens on their rows and attends to all that their slots hold;
* ``selected_attention_update`` attends to the pages that can matter most to each token.

A model trained with ``mixers.window_attention`` whose window is as long as the sequence is served by
them.  A step of a server, for chunks of one or more tokens per slot (or a packed chunk with
``cu_seqlens``, in which slots may bring none)::

    rows = paged.page_tables_update(tables, lengths, pool, tokens=T, page=page)    # once
    for layer in layers:
        output = paged.paged_attention_update(q, k, v, layer.key_pages, layer.value_pages,
                                              tables, rows, lengths)
    lengths += T

Layouts, dtypes and head widths are those of the mixers: dense ``(slots, T, heads, width)`` or
``(N, heads, width)`` with device ``cu_seqlens``; heads of keys and values shared by groups of query
heads; float32, float16 and bfloat16, widths 1 to 128.  Nothing here has a backward (inputs that ask
for one are refused), and everything can be recorded into a HIP graph.  What a call changes (tables and
pool, pages and bounds) shares no memory with what it reads, and gets a new version.  Results do not
depend on the order in which blocks run.

Nothing that is on the device is looked at by the host: invalid ``cu_seqlens`` make every output NaN
and change nothing, and numbers that are no page are never followed.  Tokens that see a key or a
value that is not finite may have outputs that are not, in one column or in all; the others keep every
bit of theirs.  In float32 a magnitude of ``2**128 - 2**119`` (3.396e38) or more counts as not finite,
and in every type sums of weights times values that pass float32's range are.  What no token was put on
is never read, but for padding among the queries of ``selected_attention_update``, whose outputs are
unspecified.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import BUILD_CAPABILITIES
from .mixers import _fake_output, _integer, _number, _unavailable

__all__ = [
    "page_tables_release",
    "page_tables_update",
    "paged_attention_update",
    "selected_attention_update",
]


# ---------------------------------------------------------------------------
# shape functions for FakeTensor / torch.compile tracing
# ---------------------------------------------------------------------------

def _register_fakes() -> None:
    register = torch.library.register_fake

    @register("rosa_soft::page_tables_update")
    def _(tables, lengths, pool, cu_seqlens, tokens, page):
        shape = (tables.shape[0], tokens) if cu_seqlens is None else (tokens,)
        return tables.new_empty(shape, dtype=torch.int64)

    @register("rosa_soft::page_tables_release")
    def _(tables, lengths, keep, pool, page):
        return None

    @register("rosa_soft::paged_attention_update")
    def _(query, key, value, key_pages, value_pages, tables, rows, lengths, cu_seqlens, scale=None):
        return _fake_output(query, value)

    @register("rosa_soft::paged_attention_update_bounds")
    def _(query, key, value, key_pages, value_pages, key_bounds, tables, rows, lengths, cu_seqlens,
          scale=None):
        return _fake_output(query, value)

    @register("rosa_soft::selected_attention_update")
    def _(query, key, value, key_pages, value_pages, key_bounds, tables, rows, lengths, cu_seqlens,
          count, scale=None):
        return _fake_output(query, value)


if BUILD_CAPABILITIES.rosa_soft_cuda:
    _register_fakes()
    _tables_update = torch.ops.rosa_soft.page_tables_update.default
    _tables_release = torch.ops.rosa_soft.page_tables_release.default
    _paged_update = torch.ops.rosa_soft.paged_attention_update.default
    _paged_update_bounds = torch.ops.rosa_soft.paged_attention_update_bounds.default
    _selected_update = torch.ops.rosa_soft.selected_attention_update.default
else:
    _tables_update = _tables_release = _paged_update = _paged_update_bounds = _unavailable
    _selected_update = _unavailable


# ---------------------------------------------------------------------------
# tables
# ---------------------------------------------------------------------------

def page_tables_update(tables: Tensor, lengths: Tensor, pool: Tensor,
                       cu_seqlens: Optional[Tensor] = None, *, tokens: int, page: int) -> Tensor:
    """Pages for the new tokens of every slot, and the rows that the tokens lie on.

    ``tables`` is int32 ``(slots, columns)``, up to 8192 slots: position ``p`` of a slot lies on page
    ``tables[slot, p // page]``, a number outside ``[0, pages)`` (-1, say) is no page.  ``pool`` is
    int32 ``(pages + 1,)``: ``pool[0]`` pages are free, and ``pool[1 : 1 + pool[0]]`` is a stack of
    their numbers; a fresh one is ``torch.arange(-1, pages)`` with ``pool[0] = pages``.
    ``lengths`` is int32 ``(slots,)``, the tokens that each slot has seen, and is left to the caller
    to advance.  ``page`` is a power of two from 16 to 256.  The new tokens are ``tokens`` for each
    slot, or with ``cu_seqlens`` (``slots + 1`` offsets) ``tokens`` packed ones in all.

    The columns that the new tokens are the first to reach take pages from the top of the stack, in
    the order of slots; where there are no more they become -1.  ``tables`` and ``pool`` are changed
    in place.  Returns int64 ``(slots, tokens)`` or ``(tokens,)``: the row of each new token,
    ``page_number * page + position % page``, or -1 for one that has no page.  All of it happens on
    the device, and can be recorded into a graph; a server that must not run out of pages reads
    ``pool[0]`` before it admits a request.  Invalid ``cu_seqlens`` change nothing, and every row
    is -1.

    Which columns are new follows from ``lengths`` alone, whatever they held before.  So of a step that
    ran out of pages, or whose tokens are not all kept (padding, rejected drafts), the rest is given back
    before the next one, ``page_tables_release(tables, lengths + new, lengths + kept, pool, page=page)``
    with the tokens that it asked for and those that stay.  Otherwise the next step takes pages for the
    same columns again and those that they had are lost, and columns that got none stay without once
    ``lengths`` has passed them.
    """

    return _tables_update(tables, lengths, pool, cu_seqlens, _integer("tokens", tokens),
                          _integer("page", page))


def page_tables_release(tables: Tensor, lengths: Tensor, keep: Tensor, pool: Tensor, *,
                        page: int) -> None:
    """Give the pages behind the first ``keep`` tokens of every slot back to the pool.

    ``keep`` is int32 ``(slots,)``: 0 for a request that ended, less than ``lengths`` for one whose
    drafted tokens were rejected, ``lengths`` (or more) for the others.  Their entries become -1 and
    their pages lie on top of the stack, the first slot's first page uppermost, so that a release
    takes back an update.  Entries that are no page are passed over, and so are pages for which the
    pool has no place.  ``lengths`` is left to the caller.

    A page in several rows of ``tables`` goes back with the last of them: while the first ``keep`` tokens
    of any slot lie on it (up to ``lengths``) it stays, and of several slots that give it back in one call
    the last one does.  A prompt that is kept for later requests has a slot of its own that brings no
    tokens.
    """

    _tables_release(tables, lengths, keep, pool, _integer("page", page))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def paged_attention_update(query: Tensor, key: Tensor, value: Tensor, key_pages: Tensor,
                           value_pages: Tensor, tables: Tensor, rows: Tensor, lengths: Tensor,
                           cu_seqlens: Optional[Tensor] = None, *,
                           key_bounds: Optional[Tensor] = None,
                           scale: Optional[float] = None) -> Tensor:
    """New tokens of every slot over all that the slot holds on its pages; no backward.

    ``query`` is ``(slots, T, H, D)``, or ``(N, H, D)`` with ``cu_seqlens`` of ``slots + 1`` offsets.
    ``key_pages`` and ``value_pages`` are contiguous ``(pages, Hkv, page, width)`` of the inputs'
    dtype, shared by all slots; ``tables`` and ``lengths`` are those of ``page_tables_update``, and
    ``rows`` (int64, one for each new token) what it returned.  The new tokens are put on their rows,
    and each attends to the positions of its slot up to its own.  ``lengths`` is left to the caller,
    who advances it once for all layers of a model.  Returns the outputs of the new tokens.

    With ``key_bounds`` (contiguous ``(pages, Hkv, 2, D)`` of the inputs' dtype) the least and the
    largest element of each column of the keys on a page are kept up to date, for
    ``selected_attention_update``.

    A new token whose row is negative (padding) is not stored, and has no part in the bounds; in this
    call the new tokens behind it see it like the others, so padding goes behind the real tokens.
    Rejected tokens may leave the bounds of their page wider than its keys.
    A token that sees a position without a page has NaN as its output.
    Slots may share pages as long as nobody writes to them (a prompt in common: the tables begin with
    the same numbers); a page that is written belongs to one slot, and no two tokens of a call to the
    same row.
    """

    scale = _number("scale", scale)
    if key_bounds is None:
        return _paged_update(query, key, value, key_pages, value_pages, tables, rows, lengths,
                             cu_seqlens, scale)
    return _paged_update_bounds(query, key, value, key_pages, value_pages, key_bounds, tables, rows,
                                lengths, cu_seqlens, scale)


def selected_attention_update(query: Tensor, key: Tensor, value: Tensor, key_pages: Tensor,
                              value_pages: Tensor, key_bounds: Tensor, tables: Tensor,
                              rows: Tensor, lengths: Tensor, cu_seqlens: Optional[Tensor] = None, *,
                              count: int, scale: Optional[float] = None) -> Tensor:
    """``paged_attention_update`` over the pages that can matter most to each token.

    A token sees, for each head of keys, its own page up to itself, and of the earlier pages the
    ``count`` (1 to 1024) with the largest ``sum_d max(q_d low_d, q_d high_d)``, the most that a key
    within a page's bounds can score, for any query head of the group: ties go to the first page,
    and a sum that is not a number ranks above all others.  The sums are formed in 64 bits.
    ``key_bounds`` must be those of the keys on the pages: kept by every update from the first token
    on, in whatever state the memory was before.  Padding goes behind the real tokens of its slot: a
    token behind one that is not stored is unspecified.
    """

    return _selected_update(query, key, value, key_pages, value_pages, key_bounds, tables, rows,
                            lengths, cu_seqlens, _integer("count", count), _number("scale", scale))
