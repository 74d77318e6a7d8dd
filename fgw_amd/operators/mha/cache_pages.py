"""Pages of the paged cache: hand out, fork, free, compact and copy (no reference counterpart: the
reference's operator reads a block table that its caller keeps).

The books of a pool are three int32 tensors on the GPU, changed in place:

  refs  [pages]        rows that hold each page; 0: the page is free
  table [rows, width]  page ids of each row, the block table of the attention entries; -1: none
  lens  [rows]         cached tokens of each row, the attention entries' cache_seqlens

Row r holds the pages table[r, : ceil(lens[r] / page_size)]; new_books makes empty books. Pools are
the K/V tensors [pages * page_size, ...] of all layers, contiguous and of any dtype, whose pages
share the ids; while gradients are recorded none may require one. Every decision is made on the GPU,
lowest free page first and rows in order, so that the results are the same on every run and no call
waits for the device: counts of what was refused come back as int32 tensors. Books that were changed
by hand must stay consistent (every held page counted in refs, and a partly filled last page held by
its row alone). Books, lists and pools of a call share no memory with each other (but lens may be
its own counts).
"""
from __future__ import annotations

from collections import namedtuple

import torch

from fgw_amd import _lib

_kv = _lib.load_kv_module()

PageBooks = namedtuple("PageBooks", "refs table lens")


def new_books(pages, rows, width, device="cuda") -> PageBooks:
    """Books of an empty pool."""
    if min(pages, rows, width) <= 0:
        raise ValueError("positive pages, rows and table width required")
    return PageBooks(torch.zeros(pages, dtype=torch.int32, device=device),
                     torch.full((rows, width), -1, dtype=torch.int32, device=device),
                     torch.zeros(rows, dtype=torch.int32, device=device))


def reserve_rows(refs, table, lens, counts, page_size):
    """Grow row r by counts[r] tokens (int32 [rows]): lens[r] += counts[r], with the pages for them.

    A row whose count is negative or would pass width * page_size tokens stays as it is, and so
    does one that needs pages where those needed up to and with it are more than the free ones.
    Returns int32 [2]: rows refused for want of pages, rows refused for their count.
    """
    return _kv.reserve(refs, table, lens, counts, page_size)


def fork_rows(pools, refs, table, lens, parents, children, page_size):
    """Make row children[i] a copy of row parents[i] (int32 [n] each), for beams and samples.

    The whole pages are shared; a partly filled last page is copied, in every pool, to the lowest
    free page, so both rows can be written on. A pair is refused, and its child stays empty, when a
    row is out of range, when the child holds tokens, is a parent of this call or the child of an
    earlier pair, or when no page is left for it (pages go to the pairs in order). Returns int32
    [2]: pairs refused for want of pages, pairs refused for their rows.
    """
    return _kv.fork(pools, refs, table, lens, parents, children, page_size)


def free_rows(refs, table, lens, rows, page_size):
    """Empty the rows (int32 [n]): their pages lose a holder, lens 0, table entries -1. Rows out of
    range, empty ones and ones listed before are left."""
    _kv.free(refs, table, lens, rows, page_size)


def compact_pages(pools, refs, table, lens, page_size):
    """Move the live pages to the ids 0 .. L - 1, L their number, in every pool, table and refs with
    them: the i-th live page from L on goes to the i-th free page below L. What lies from L on is
    free afterwards. Returns int32 [1]: pages moved."""
    return _kv.compact(pools, refs, table, lens, page_size)


def copy_pages(pools, src, dst, page_size):
    """Copy page src[i] to page dst[i] (int32 [n] each) in every pool. Pairs with an id outside the
    pools are skipped. No page may be a destination twice, or a destination and a source."""
    if not pools:
        raise ValueError("at least one pool required")
    if page_size <= 0 or pools[0].shape[0] == 0 or pools[0].shape[0] % page_size:
        raise ValueError("positive page size and whole pool pages required")
    _kv.copy(pools, src, dst, pools[0].shape[0] // page_size, page_size)
