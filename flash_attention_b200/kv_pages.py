"""Pages of a KV cache: which sequence has which, and copying them.

A page table is an argument of every call that reads or fills a paged cache (:func:`flash_attn_fp4_func`, :func:`append_kv_fp8`,
:func:`flash_attn_fp8_cache_func`, :func:`flash_attn_fp8_blocks_func`).  Here it is kept on the device: sequences grow, end and are forked
(beams, several samples of one prompt) without the host looking on, so a serving step with its book-keeping can be captured in a graph.  The caches of all
layers share one table; what has to be copied comes back as pairs of pages for :func:`copy_kv_pages` of each.  A step of a loop:

    pages, held = fork_kv_pages(pages, held, parents)          # beams: rows go on from the beams they were chosen from
    pairs = resize_kv_pages(pages, held, held + 1, granted=room)           # room for a token; rows that end: wanted 0
    for cache in layers: copy_kv_pages(cache, pairs)
    for cache in layers: append_kv_fp8(cache, k, v, held, page_table=pages.table, seqused_new=room - held) ...
    held.copy_(room)

Where the pool is sure to have a page for everybody ``granted`` is what was wanted, and may be left out.

No counterpart in the reference, whose callers make page tables on the host.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .fp8_cache import FP8KVCache


@dataclass
class KVPages:
    """Who has which page of a pool.

    table      (B, pages_per_seq) int32, contiguous: pages of a sequence, in order; -1 where it has none (-2^31 + page: see :func:`resize_kv_pages`)
    refs       (num_pages,) int32, contiguous: how many entries name a page; 0: it is free
    page_size  tokens of a page, as in the caches

    Calls that change the same refs or table must not overlap (one stream, or events between them).
    """
    table: torch.Tensor
    refs: torch.Tensor
    page_size: int

    @classmethod
    def empty(cls, num_seqs: int, pages_per_seq: int, num_pages: int, page_size: int, device=None) -> "KVPages":
        """Sequences without pages, and a pool whose pages are all free."""
        device = torch.device("cuda") if device is None else torch.device(device)
        return cls(torch.full((num_seqs, pages_per_seq), -1, dtype=torch.int32, device=device),
                   torch.zeros(num_pages, dtype=torch.int32, device=device), page_size)


def resize_kv_pages(pages: KVPages, held: torch.Tensor, wanted: torch.Tensor, granted: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Pages for ``wanted[b]`` tokens for every sequence, of which it holds ``held[b]``; returns the pages to copy, (B, 2) int32 (from, to), -1 where
    there is none (:func:`copy_kv_pages`).  ``pages`` is changed in place; held and wanted (B,) int32 are not.

    A sequence keeps the pages of its first min(held, wanted) tokens and gives back those behind (wanted 0: all of them; less than held: drafted tokens that
    were not accepted), then gets free ones, the lowest first, sequences in order.  Where it grows and its next token goes into a page that already holds some of its tokens and
    belongs to others too, it gets a copy of that page; of the sequences that would write to it the last keeps it, if nobody else has it.  Pages given back may
    be given out by the same call, and what pages behind ``held`` contained is lost.

    Where no page is left, :func:`check_status` raises, and what a sequence holds stays as it is:

    * an entry that should have got a page is -1 (what is appended there is left out);
    * a copy is not made: the sequence goes on sharing the page, and neither it nor the one that was to keep the page gets to write there.  With ``granted`` their entries stay and can be
      read; without it they become -2^31 + page, which the calls on a cache take for no page (nothing is appended or read there, and they report it), until the next call of this function
      that has a page or does not let them grow;
    * a sequence that has no page for some of the tokens it keeps (they were left out before) gets nothing until it is cut in front of them: what they were is lost.  Without ``granted``
      the page that its next token would go to is marked in the same way.

    ``granted`` (B,) int32, overlapping none of the others, is written: the lengths that may be appended up to.  That is ``wanted`` if nothing was missing, else the tokens in front
    of the first entry without a page, or ``held`` where a copy was not made; append with ``seqused_new=granted - held`` and go on with it as the next held.  The same call works once
    there are pages again.

    One launch, no synchronisation; can be captured in a graph.  At most 4096 sequences.  Where lengths or entries lie outside the table or the pool they are cut
    or dropped, and :func:`check_status` raises.
    """
    return _lib.host().resize_pages(pages.table, pages.refs, pages.page_size, held, wanted, granted)


def fork_kv_pages(pages: KVPages, held: torch.Tensor, parents: torch.Tensor,
                  out: Optional[Tuple[KVPages, torch.Tensor]] = None) -> Tuple[KVPages, torch.Tensor]:
    """Sequences that go on from others: row i of the result is row ``parents[i]`` of ``pages`` as far as it holds tokens (-1: an empty row), together with
    its held.  Rows that nobody goes on from are given back.

    ``parents`` (rows,) int32: any number of rows, the same parent as often as wanted.  The pages are shared, none is copied (:func:`resize_kv_pages` does that for
    what is written to).  ``refs`` is changed in place and belongs to the result; the old table is worth nothing afterwards.  ``out``: what an earlier call returned for as many
    rows, with the same refs, to be written over; it must not be ``pages`` itself (two tables that take turns).

    One launch, no synchronisation; can be captured in a graph.  A parent outside the table gives an empty row, and :func:`check_status` raises.
    """
    table, into = (None, None) if out is None else (out[0].table, out[1])
    if out is not None and (out[0].refs.data_ptr() != pages.refs.data_ptr() or out[0].page_size != pages.page_size):
        raise ValueError("out must have the refs and the page_size of pages")
    table, into = _lib.host().fork_pages(pages.table, pages.refs, pages.page_size, held, parents, table, into)
    return (KVPages(table, pages.refs, pages.page_size), into) if out is None else out


def compact_kv_pages(pages: KVPages) -> Tuple[torch.Tensor, torch.Tensor]:
    """Moves the pages in use to the front of the pool: returns the pages to copy, (num_pages // 2, 2) int32 (from, to), -1 behind the last, and how many are in use, (1,)
    int32.  ``pages`` is changed in place; the table must be the only one that names pages of the pool.

    With n pages in use the i-th of those numbered n or above goes to the i-th free one below; what lies at n and above is free afterwards (the pool may be cut there once
    :func:`copy_kv_pages` has run).  A table without rows is refused.  One launch, no synchronisation; can be captured in a graph.
    """
    return _lib.host().compact_pages(pages.table, pages.refs, pages.page_size)


def copy_kv_pages(cache: Union[FP8KVCache, torch.Tensor, Sequence], pairs: torch.Tensor) -> None:
    """Copies page ``pairs[i, 0]`` to page ``pairs[i, 1]`` for every i; pairs (n, 2) int32 with a negative number are none.

    ``cache``: an :class:`FP8KVCache` (its index too), a tensor whose first dimension is that of pages (any type, strided as a pool may be), or a sequence of
    such (all of one number of pages).  No page may be written twice, or both read and written, in one call: what the other calls return has no such pairs.

    One launch for eight tensors (from 64 MB on two, if pages of some lie in one piece and of others not), no synchronisation; can be captured in a graph.  Pairs outside the pool are left out, and :func:`check_status` raises.
    """
    if isinstance(cache, FP8KVCache):
        tensors = cache.tensors()
    elif isinstance(cache, torch.Tensor):
        tensors = (cache,)
    else:
        tensors = tuple(t for c in cache for t in (c.tensors() if isinstance(c, FP8KVCache) else (c,)))
    _lib.host().copy_pages(pairs, tensors)
