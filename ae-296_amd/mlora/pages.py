"""Page tables of a cache that live on the device and share pages: what a serving loop changes from step to step without waiting for it.

    pages = KVPages(cache, n_req, max_pages)
    pages.resize(want)                              # new lengths: pages handed out, given back, copied where they are shared
    batch = KVBatch(pages.grown, pages.lens - 1, pages.table, ...)      # one new token a row, for the rows that could be served
    ...
    pages.fork(parent)                              # beams, or more answers to one prompt

Row r of `table` names the pages of request r's own `lens[r]` tokens; `refs` counts the entries that name each page.  A step that plans attention does
so after these calls.  They launch on ``torch.cuda.current_stream()``, allocate nothing, do not synchronise and may be captured; calls on one object are
ordered on one stream, graphs that were captured with it included.  The counterpart of the reference's MemoryManager
(``lightllm/common/mem_manager.py:4-111``) and ReqManager (``req_manager.py:3-36``).
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np
import torch

from . import _ext
from .attention import KVCache


class KVPages:
    """Tables for `n_req` requests of up to `max_pages` pages each, over `n_pages` pages taken from the cache (by default all it has
    free).  `state` holds all of it (int32): a copy of it is a snapshot, which may be copied back until the next ``take``, ``give_back`` or
    ``compact``; what was written to the cache meanwhile stays written."""

    def __init__(self, cache: KVCache, n_req: int, max_pages: int, n_pages: Optional[int] = None):
        at = (C.c_int64 * _ext.PAGES_LAYOUT_WORDS)()
        _ext.check(_ext.lib().mlora_pages_layout(n_req, max_pages, cache.n_pages, at))
        if max_pages * cache.page_tokens > 1 << 30:
            raise ValueError("max_pages * page_tokens may be 2^30 at most")
        _, table, lens, refs, failed, live, words, scratch = at
        self.cache, self.n_req, self.max_pages = cache, n_req, max_pages
        self.state = torch.zeros(words, dtype=torch.int32, device=cache.device)
        self.scratch = torch.zeros(scratch, dtype=torch.int32, device=cache.device)
        # a byte a page
        self._free, self._managed = (x[:table].view(torch.uint8)[:cache.n_pages] for x in (self.state, self.scratch))
        self.table = self.state[table:lens].view(n_req, max_pages)
        self.lens, self.refs = self.state[lens:refs], self.state[refs:failed]
        self.failed = self.state[failed:live]          # rows that resize or fork could not serve, added up until it is cleared
        self.live = self.state[live:words]             # pages in use, as of the last compact
        # r where the last resize made row r longer, else -1 (all of them after fork and adopt); not part of a snapshot
        self.grown = self.scratch[table:table + n_req]
        self.grown.fill_(-1)
        self.table.fill_(-1)
        self.take(cache.free_pages if n_pages is None else n_pages)

    def take(self, n: int) -> None:
        """n more pages of the cache."""
        ids = torch.from_numpy(np.array(self.cache.allocate(n), np.int64)).to(self.state.device)
        self._managed[ids] = 1
        self._free[ids] = 1

    def give_back(self) -> int:
        """Gives the cache the pages behind the last one in use (all that are free, after ``compact``) and returns how many.
        Waits for the device."""
        managed, free = self._managed.cpu().numpy().astype(bool), self._free.cpu().numpy().astype(bool)
        used = np.flatnonzero(managed & ~free)
        ids = np.flatnonzero(free)
        ids = ids[ids > (used[-1] if len(used) else -1)]
        gone = torch.from_numpy(ids).to(self.state.device)
        self._managed[gone] = 0
        self._free[gone] = 0
        self.cache.release(ids.tolist())
        return len(ids)

    def adopt(self, table: torch.Tensor, lens: torch.Tensor) -> None:
        """Tables and lengths from elsewhere (int32 [n_req, max_pages] and [n_req]) in place of the present ones; pages that several rows
        name are shared, and what lies behind a row's last page does not count.  Waits for the device."""
        if tuple(table.shape) != (self.n_req, self.max_pages) or tuple(lens.shape) != (self.n_req,):
            raise ValueError(f"expected a table [{self.n_req}, {self.max_pages}] and {self.n_req} lengths")
        M, N, device = self.max_pages, self.cache.n_pages, self.state.device
        table, lens = table.to(device), lens.to(device)
        n, column = lens.long(), torch.arange(M, device=device)
        held = column < ((n + self.cache.page_tokens - 1) // self.cache.page_tokens)[:, None]
        # entries that do not count: places of their own behind the last page, a column each
        at = torch.where(held, table, N + column)
        exists = (at >= 0) & (at < N + M)
        at = torch.where(exists, at, N + column)
        known = torch.cat((self._managed.bool(), torch.ones(M, dtype=torch.bool, device=device)))
        in_order = torch.sort(at, 1)[0]
        fine = torch.stack((((n >= 0) & (n <= M * self.cache.page_tokens)).all(), exists.all() & (known[at] | ~held).all() & ((at < N) == held).all(),
                            (in_order[:, 1:] != in_order[:, :-1]).all())).tolist()
        if not fine[0]:
            raise ValueError(f"lengths must be in 0..{M * self.cache.page_tokens}")
        if not fine[1]:
            raise ValueError("a row names a page that is not among the managed ones")
        if not fine[2]:
            raise ValueError("a row names a page twice")
        refs = torch.zeros(N + M, dtype=torch.int32, device=device)
        refs.index_add_(0, at.view(-1), torch.ones_like(at, dtype=torch.int32).view(-1))
        self.table.copy_(torch.where(held, at, -1))
        self.lens.copy_(n)
        self.refs.copy_(refs[:N])
        self._free.copy_(self._managed.bool() & (self.refs == 0))
        self.grown.fill_(-1)

    def resize(self, want: torch.Tensor) -> None:
        """Rows' new lengths, int32 [n_req] on the device and not `lens` itself (negative: as it is; 0 gives all pages back).  Shorter
        rows give pages back first; then longer rows, in their order, get the lowest free ids.  A longer row that will write on a page other
        rows name as well gets its own copy of what that holds, in all layers - the last of them keeps the page if all of them do.  A row
        that does not fit keeps its length and pages and counts in `failed`; so does every later one that needs a page.

        A step appends to rows that got longer and to no others, from their old length on: a row that was not served still names the page that it was
        refused a copy of, and what is appended there replaces other rows' tokens.  `grown` says which rows these are, on the device: as the ``tok_req`` of
        a batch of one token a row (the others are then left alone, their outputs zeros), or by ``grown[row]`` for several tokens a row."""
        rc = _ext.host().pages_resize(self, want)
        if rc:
            _ext.check(rc)

    def fork(self, parent: torch.Tensor) -> None:
        """Row r goes on from row parent[r]'s tokens (int32 [n_req] on the device; negative or r itself: from its own), all rows at once,
        so a permutation is one too.  Pages are shared, the last one too: ``resize`` comes before the next token is appended, and
        copies what would be written on.  A parent of n_req or more leaves the row as it is and counts in `failed`."""
        rc = _ext.host().pages_fork(self, parent)
        if rc:
            _ext.check(rc)

    def compact(self) -> None:
        """Moves the pages in use to the lowest ids, with their keys and values; `live` says how many there are.  Copies of `table` made
        before are void afterwards."""
        rc = _ext.host().pages_compact(self)
        if rc:
            _ext.check(rc)
