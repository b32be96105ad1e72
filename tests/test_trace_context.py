"""A trace's cache when it runs short: a refused step changes nothing, and prompts nobody runs give way."""
import pytest
import torch

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


def test_prompts_of_adapters_that_nobody_runs_give_way():
    """Twenty adapters, one after the other, on pages for three prompts; a prompt that comes back holds what it held."""
    c = context(8)
    first = c.advance([0], [0])
    k = c.cache.k[:, first["prefix_pages"][0]].clone()
    for a in range(1, 20):
        b = c.advance([a], [a])
        assert len(b["prefix_len"]) == 1 and b["req_prefix"] == [0]
        assert len(set(b["prefix_pages"][0]) | set(b["pages"][0])) == 3
    back = c.advance([100], [0])
    assert torch.equal(c.cache.k[:, back["prefix_pages"][0]], k)
    pages = [p for ps in c.prompts.values() for p in ps] + [p for ps in c.pages.values() for p in ps]
    assert len(set(pages)) == len(pages) and c.cache.free_pages + len(pages) == 8


def test_prompts_are_kept_while_there_is_room_and_the_last_used_stay_longest():
    c = context(10)
    p = {a: c.advance([a], [a])["prefix_pages"][0] for a in (1, 2, 3)}
    assert c.advance([7, 8], [1, 3])["prefix_pages"] == [p[1], p[3]] and set(c.prompts) == {1, 2, 3}
    c.advance([7, 8, 9], [1, 3, 4])                               # 2 was used longest ago
    assert set(c.prompts) == {1, 3, 4} and c.prompts[1] == p[1] and c.prompts[3] == p[3]


def test_a_step_lists_the_prompts_of_its_own_requests_only():
    c = context(20)
    c.advance([1, 2], [5, 6])
    b = c.advance([2, 3, 4], [6, 7, 6])
    assert b["req_prefix"] == [0, 1, 0] and b["prefix_pages"] == [c.prompts[6], c.prompts[7]] and b["prefix_len"] == [17, 17]


def test_prompts_in_use_are_not_given_back():
    c = context(8)
    c.advance([1, 2], [5, 6])
    before = state(c)
    with pytest.raises(MemoryError):
        c.advance([1, 2, 3], [5, 6, 7])
    assert state(c) == before
