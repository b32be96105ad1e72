"""A trace's cache when it runs short."""
import pytest

import mlora
from mlora.trace_driver import TraceContext


def context(pages, prompt=17):
    return TraceContext(mlora.KVCache(1, pages, 1, 64, device="cpu"), prompt, seed=3)


def state(c):
    return ({r: list(p) for r, p in c.pages.items()}, dict(c.length), {a: list(p) for a, p in c.prompts.items()}, c.cache.free_pages)


def test_a_step_that_does_not_fit_changes_nothing():
    c = context(8)
    c.advance([1, 2, 3], [5, 5, 5])
    before = state(c)
    with pytest.raises(MemoryError):
        c.advance([3, 10, 11, 12, 13, 14, 15], [5] * 7)          # 1 and 2 end, six come: six pages where three are free and two come back
    assert state(c) == before
    b = c.advance([1, 2, 3], [5, 5, 5])
    assert b["tok_pos"] == [18, 18, 18]


def test_pages_of_ended_requests_serve_the_same_step():
    c = context(6)
    c.advance([1, 2, 3, 4], [5] * 4)
    assert c.cache.free_pages == 0
    b = c.advance([4, 6, 7, 8], [5] * 4)
    assert b["tok_pos"] == [18, 17, 17, 17] and len({p for r in b["pages"] for p in r}) == 4
