"""Pages in a table that are not among the managed ones: counted and copied from, but never handed out and never moved."""
import pytest
import torch

import mlora
from gpu_common import say

pytestmark = pytest.mark.gpu


def tables(rows, n_pages=12, foreign=(0, 3, 9), max_pages=4):
    """KVPages over a cache whose pages `foreign` something else has, and rows (pages, tokens) as a state that another program wrote."""
    cache = mlora.KVCache(2, n_pages, 2, 64)
    for t in (cache.k, cache.v):
        t.copy_(torch.randn(t.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(n_pages)))
    got = cache.allocate(n_pages)
    cache.release([p for p in got if p not in foreign])
    pages = mlora.KVPages(cache, len(rows), max_pages)
    table = [list(p) + [-1] * (max_pages - len(p)) for p, _ in rows]
    refs = [sum(row.count(p) for row in table) for p in range(n_pages)]
    pages.table.copy_(torch.tensor(table))
    pages.lens.copy_(torch.tensor([n for _, n in rows]))
    pages.refs.copy_(torch.tensor(refs))
    pages._free.copy_(torch.tensor([p not in foreign and refs[p] == 0 for p in range(n_pages)]))
    return cache, pages


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("n_req, max_pages", [(2, 4), (40, 2000), (1500, 8), (1500, 50)])
def test_pages_given_back(n_req, max_pages):
    say(f"foreign pages given back {n_req} x {max_pages}")
    _, p = tables([([0, 3, 9], 48), ([3, 1], 20)] + [([], 0)] * (n_req - 2), max_pages=max_pages)
    p.resize(ints([16, 0] + [-1] * (n_req - 2)))
    assert p.refs.tolist() == [1] + [0] * 11 and p._free.nonzero().flatten().tolist() == [1, 2, 4, 5, 6, 7, 8, 10, 11]
    p.resize(ints([0, min(max_pages, 9) * 16] + [-1] * (n_req - 2)))
    assert p.table[1].tolist()[:9] == [1, 2, 4, 5, 6, 7, 8, 10, 11][:max_pages]
    p.resize(ints([0] * n_req))
    p.compact()
    assert p.live.tolist() == [0] and p._free.sum() == 9 and p.give_back() == 9


def test_pages_dropped_by_a_fork():
    say("foreign pages dropped by a fork")
    _, p = tables([([0, 9], 30), ([1], 5), ([3, 2], 17)])
    p.fork(ints([1, -1, 1]))
    assert p.refs.tolist() == [0, 3] + [0] * 10 and p._free.nonzero().flatten().tolist() == [2, 4, 5, 6, 7, 8, 10, 11]
    p.resize(ints([16, 5, 64]))
    assert p.failed.tolist() == [0] and not {0, 3, 9} & set(p.table.flatten().tolist())


def test_a_foreign_page_that_is_written_on():
    say("foreign page written on")
    cache, p = tables([([5, 9], 20), ([6, 9], 20), ([0], 3)])
    k = cache.k.clone()
    p.resize(ints([21, 21, 4]))               # row 0 copies, row 1 keeps the page, nobody shares row 2's
    assert p.table.tolist() == [[5, 1, -1, -1], [6, 9, -1, -1], [0, -1, -1, -1]] and p.refs.tolist() == [1, 1, 0, 0, 0, 1, 1, 0, 0, 1, 0, 0]
    assert torch.equal(cache.k[:, 1, :, :4], k[:, 9, :, :4])
    p.compact()                               # managed and in use: 1, 5, 6 -> 1, 2, 4; the others stay
    assert p.table.tolist() == [[2, 1, -1, -1], [4, 9, -1, -1], [0, -1, -1, -1]] and p.live.tolist() == [3]
    assert torch.equal(cache.k[:, 2], k[:, 5]) and torch.equal(cache.k[:, 4], k[:, 6]) and torch.equal(cache.k[:, 9], k[:, 9]) and torch.equal(cache.k[:, 0], k[:, 0])
