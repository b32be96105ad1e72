"""Page tables of a cache that live on the device and share pages: what a serving loop changes from step to step without waiting for it.

    pages = KVPages(cache, n_req, max_pages)
    pages.resize(want)                              # new lengths: pages handed out, given back, copied where they are shared
    batch = KVBatch(tok_req, tok_pos, pages.table, ...)
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
    """Tables for `n_req` requests of up to `max_pages` pages each, over `n_pages` pages taken from the cache (by default all it has free).  `state` holds all of
    it (int32): a copy of it is a snapshot, and copying that back restores it, but not what was written to the cache meanwhile."""

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
        self.table.fill_(-1)
        self.take(cache.free_pages if n_pages is None else n_pages)

    def take(self, n: int) -> None:
        """n more pages of the cache."""
        ids = torch.tensor(self.cache.allocate(n), dtype=torch.long, device=self.state.device)
        self._managed[ids] = 1
        self._free[ids] = 1

    def give_back(self) -> int:
        """Gives the cache the pages behind the last one in use (all that are free, after ``compact``) and returns how many.  Waits for the device."""
        managed, free = self._managed.cpu().numpy().astype(bool), self._free.cpu().numpy().astype(bool)
        used = np.flatnonzero(managed & ~free)
        ids = np.flatnonzero(free)
        ids = ids[ids > (used[-1] if len(used) else -1)]
        gone = torch.from_numpy(ids).to(self.state.device)
        self._managed[gone] = 0
        self._free[gone] = 0
        self.cache.release(ids[::-1].tolist())
        return len(ids)

    def adopt(self, table: torch.Tensor, lens: torch.Tensor) -> None:
        """Tables and lengths from elsewhere (int32 [n_req, max_pages] and [n_req]) in place of the present ones; pages that several rows name are shared, and what
        lies behind a row's last page does not count.  Waits for the device."""
        if tuple(table.shape) != (self.n_req, self.max_pages) or tuple(lens.shape) != (self.n_req,):
            raise ValueError(f"expected a table [{self.n_req}, {self.max_pages}] and {self.n_req} lengths")
        n = lens.cpu().numpy().astype(np.int64)
        if (n < 0).any() or (n > self.max_pages * self.cache.page_tokens).any():
            raise ValueError(f"lengths must be in 0..{self.max_pages * self.cache.page_tokens}")
        held = torch.arange(self.max_pages, device=table.device) < torch.from_numpy(-(-n // self.cache.page_tokens)).to(table.device)[:, None]
        ids = table[held].long()
        if ids.numel() and (int(ids.min()) < 0 or int(ids.max()) >= self.cache.n_pages or not bool(self._managed.to(ids.device)[ids].all())):
            raise ValueError("a row names a page that is not among the managed ones")
        pairs = torch.sort(held.nonzero()[:, 0] * self.cache.n_pages + ids)[0]
        if bool((pairs[1:] == pairs[:-1]).any()):
            raise ValueError("a row names a page twice")
        refs = torch.bincount(ids, minlength=self.cache.n_pages).to(torch.int32)
        self.table.copy_(table.masked_fill(~held, -1))
        self.lens.copy_(lens)
        self.refs.copy_(refs)
        self._free.copy_(self._managed.bool() & (self.refs == 0))

    def resize(self, want: torch.Tensor) -> None:
        """Rows' new lengths, int32 [n_req] on the device (negative: as it is; 0 gives all pages back).  Shorter rows give pages back first; then longer rows, in
        their order, get the lowest free ids.  A longer row that will write on a page other rows name as well gets its own copy of what that
        holds, in all layers - the last of them keeps the page if all of them do.  A row that does not fit keeps its length and pages and counts in
        `failed`; so does every later one that needs a page."""
        rc = _ext.host().pages_resize(self, want)
        if rc:
            _ext.check(rc)

    def fork(self, parent: torch.Tensor) -> None:
        """Row r goes on from row parent[r]'s tokens (int32 [n_req] on the device; negative or r itself: from its own), all rows at once, so a permutation is one
        too.  Pages are shared until one of the rows writes on them (``resize``).  A parent of n_req or more counts in `failed`."""
        rc = _ext.host().pages_fork(self, parent)
        if rc:
            _ext.check(rc)

    def compact(self) -> None:
        """Moves the pages in use to the lowest ids, with their keys and values; `live` says how many there are.  Tables made before (plans, copies of `table`) are
        void afterwards."""
        rc = _ext.host().pages_compact(self)
        if rc:
            _ext.check(rc)
