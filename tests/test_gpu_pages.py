"""Page tables on the device against the sequential model: every table, length and count, and every key and value, after every call."""
import numpy as np
import pytest
import torch

import mlora
from gpu_common import say
from pages_ref import Tables

pytestmark = pytest.mark.gpu


class Pair:
    """A KVPages and the model of it, over a cache whose every element differs."""

    def __init__(self, n_req, max_pages, n_pages, P=16, layers=2, kv_heads=2, D=64, dtype=torch.float16, held_back=(), taken=None):
        say(f"pages n_req={n_req} max_pages={max_pages} n_pages={n_pages} P={P} layers={layers}")
        self.cache = mlora.KVCache(layers, n_pages, kv_heads, D, page_tokens=P, dtype=dtype)
        g = torch.Generator(device="cuda").manual_seed(n_pages)
        for t in (self.cache.k, self.cache.v):
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))
        if held_back:                    # pages that something else has
            got = self.cache.allocate(n_pages)
            self.cache.release([p for p in got if p not in held_back])
        self.pages = mlora.KVPages(self.cache, n_req, max_pages, taken)
        managed = [p for p in range(n_pages) if p not in held_back]
        if taken is not None:
            managed = self.pages._managed.nonzero().flatten().tolist()
        self.model = Tables([[] for _ in range(n_req)], [0] * n_req, managed, n_pages, P, max_pages)
        self.k, self.v = self.cache.k.clone(), self.cache.v.clone()

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def check(self, what=""):
        m, p = self.model, self.pages
        assert p.lens.tolist() == m.lens, what
        assert p.table.tolist() == m.table(), what
        assert p.refs.tolist() == m.refs(), what
        assert p.failed.tolist() == [m.failed], what
        refs = m.refs()
        assert p._free.nonzero().flatten().tolist() == [i for i in m.managed if refs[i] == 0], what
        assert torch.equal(self.cache.k, self.k) and torch.equal(self.cache.v, self.v), what

    def resize(self, want, check=True):
        for a, b, n in self.model.resize(want):
            for t in (self.k, self.v):
                t[:, b, :, :n] = t[:, a, :, :n]
        self.pages.resize(self.ints(want))
        if check:
            self.check(f"resize {want}")

    def fork(self, parent):
        self.model.fork(parent)
        self.pages.fork(self.ints(parent))
        self.check(f"fork {parent}")

    def compact(self):
        moves = self.model.compact()
        for t in (self.k, self.v):
            old = t.clone()
            for a, b in moves:
                t[:, b] = old[:, a]
        self.pages.compact()
        self.check("compact")
        assert self.pages.live.tolist() == [sum(n > 0 for n in self.model.refs())]


def test_lengths_at_the_ends_of_pages():
    p = Pair(6, 8, 40)
    for want in ([1, 16, 17, 0, 128, 31], [1, 16, 17, 0, 128, 31], [2, 17, 16, 1, 127, 32], [0, 33, 15, -1, 112, -7], [0] * 6, [128, 0, 0, 128, 0, 0], [-1] * 6):
        p.resize(want)


def test_a_page_that_others_hold_is_copied_before_it_is_written():
    p = Pair(4, 4, 20, layers=3)
    p.resize([21, 0, 0, 0])
    p.fork([-1, 0, 0, 3])
    p.resize([22, -1, 40, -1])            # one holder stays: both writers copy
    p.resize([23, 22, 41, 5])             # the last one alone
    p.fork([1, 1, 1, 1])
    p.resize([23, 23, 23, 23])            # all write: the last keeps the page


def test_a_shared_page_in_the_middle_after_taking_tokens_back():
    p = Pair(3, 6, 30)
    p.resize([70, 0, 0])
    p.fork([0, 0, 0])
    p.resize([-1, 20, 36])                # ends inside pages that row 0 still holds
    p.resize([71, 21, 48])
    p.resize([0, 33, 49])
    p.resize([64, 64, 64])                # full pages: nothing to copy


@pytest.mark.parametrize("want", [[40, 40, 40], [200, 16, 16], [16, 200, 16], [17, 1, 300], [129, 1, 1], [1 << 30, 2, 2 ** 31 - 1]])
def test_rows_that_do_not_fit(want):
    p = Pair(3, 8, 7)
    p.resize([16, 15, 31])
    p.resize(want)
    p.resize([17, 16, 32])


def test_a_row_that_keeps_a_page_waits_for_those_that_copy_it():
    """Without room for the copy, no row may write on the shared page."""
    p = Pair(3, 4, 2)
    p.resize([20, 0, 0])
    p.fork([0, 0, -1])
    p.resize([21, 21, 0])
    assert p.model.failed == 2 and p.model.lens == [20, 20, 0]
    p.resize([0, 21, 0])                  # alone now
    assert p.model.lens == [0, 21, 0]


def test_pages_given_back_in_a_call_are_handed_out_in_it():
    p = Pair(4, 4, 8)
    p.resize([64, 64, 0, 0])
    p.resize([0, 17, 64, 32])
    p.resize([0, 0, 0, 0])


def test_forks_are_made_at_once():
    p = Pair(5, 4, 30)
    p.resize([10, 20, 33, 64, 0])
    p.fork([1, 2, 0, 4, 3])               # a permutation
    p.fork([0, 1, 2, 3, 4])
    p.fork([-1, 0, 1, 2, 3])
    p.fork([5, 7, -3, 2 ** 31 - 1, 0])    # parents that do not exist
    p.fork([4, 4, 4, 4, 4])


def test_a_fork_takes_what_only_the_forked_row_had():
    p = Pair(2, 4, 10)
    p.resize([64, 30])
    p.fork([1, 0])
    p.fork([1, 1])
    p.resize([0, 0])


def test_compact_moves_what_is_beyond():
    p = Pair(6, 6, 50)
    p.resize([90, 1, 33, 60, 17, 0])
    p.resize([0, 1, 20, 0, 17, 90])
    p.fork([-1, -1, -1, 2, -1, -1])
    p.resize([-1, -1, -1, -1, 0, -1])
    p.compact()
    p.compact()
    p.resize([16, 40, 25, 25, 3, 70])
    p.resize([0] * 6)
    p.compact()


def test_pages_that_are_not_its_own_stay():
    back = {0, 1, 7, 20, 38, 39}
    p = Pair(4, 8, 40, held_back=back)
    p.resize([100, 50, 20, 0])
    p.resize([0, 50, 20, 60])
    p.compact()
    p.resize([128, 128, 128, 127])
    p.resize([128, 128, 128, 128])
    assert not back & {i for row in p.model.rows for i in row}


def test_pages_are_taken_and_given_back():
    p = Pair(2, 8, 30, taken=6)
    assert p.cache.free_pages == 24
    p.resize([64, 33])
    assert p.model.failed == 1
    p.pages.take(4)
    p.model.managed = p.pages._managed.nonzero().flatten().tolist()
    p.resize([64, 33])
    p.resize([0, -1])
    p.compact()
    assert p.pages.give_back() == 7 and p.cache.free_pages == 27
    p.model.managed = p.model.managed[:3]
    p.resize([1, 48])
    assert p.model.failed == 2 and p.pages.give_back() == 0
    p.resize([0, 0])
    assert p.pages.give_back() == 3 and p.cache.free_pages == 30
    assert p.cache.allocate(3) == [0, 1, 2]


def test_adopted_tables():
    p = Pair(3, 4, 20)
    p.pages.adopt(p.ints([[5, 9, 19, 3], [5, 9, 7, 7], [-1, 2, 2, 2]]), p.ints([64, 40, 0]))
    p.model = Tables([[5, 9, 19, 3], [5, 9, 7], []], [64, 40, 0], range(20), 20, 16, 4)
    p.check()
    p.resize([48, 41, 3])
    start = p.pages.state.clone()
    p.resize([0, 0, 0])
    p.pages.state.copy_(start)            # a snapshot
    p.model = Tables([[5, 9, 19], [5, 9, 7], [0]], [48, 41, 3], range(20), 20, 16, 4)
    p.check()
    for table, lens in (([[5, 20, 1, 1]] + [[-1] * 4] * 2, [17, 0, 0]), ([[5, 5, 1, 1]] + [[-1] * 4] * 2, [17, 0, 0]), ([[-1] * 4] * 3, [0, 1, 0]),
                        ([[-1] * 4] * 3, [0, -1, 0]), ([[0, 1, 2, 3]] * 3, [0, 65, 0])):
        with pytest.raises(ValueError):
            p.pages.adopt(p.ints(table), p.ints(lens))
    p.check()


@pytest.mark.parametrize("P, layers, kv_heads, D, dtype", [(16, 1, 1, 64, torch.float16), (32, 2, 10, 128, torch.bfloat16), (256, 1, 3, 64, torch.float16), (64, 5, 2, 128, torch.float16)])
@pytest.mark.parametrize("seed", range(3))
def test_random_steps(P, layers, kv_heads, D, dtype, seed):
    rng = np.random.default_rng(seed)
    R = int(rng.integers(1, 40))
    p = Pair(R, 5, int(rng.integers(R, 4 * R + 4)), P=P, layers=layers, kv_heads=kv_heads, D=D, dtype=dtype)
    for step in range(14):
        what = rng.integers(0, 6)
        if what == 5:
            p.compact()
        elif what == 4:
            p.fork(np.where(rng.random(R) < 0.4, rng.integers(0, R, R), -1).tolist())
        else:
            lens = np.array(p.model.lens)
            kind = rng.random(R)
            want = np.where(kind < 0.5, lens + rng.integers(0, 4, R), np.where(kind < 0.65, rng.integers(0, 5 * P + 1, R), np.where(kind < 0.75, 0, np.where(kind < 0.85, lens - 3, -1))))
            p.resize(want.tolist())


def test_more_rows_and_pages_than_a_workgroup_has_threads():
    """Sums go on from one round of 1024 rows, and of 64 * 1024 pages, to the next."""
    R, N = 2600, 150000
    p = Pair(R, 70, N, P=16, layers=1, kv_heads=1, D=64)
    rng = np.random.default_rng(0)
    p.resize((rng.integers(0, 70 * 16 + 1, R)).tolist())
    p.resize((rng.integers(0, 2, R) * rng.integers(0, 70 * 16 + 1, R)).tolist())
    p.fork(np.where(rng.random(R) < 0.5, rng.integers(0, R, R), -1).tolist())
    p.resize((np.minimum(np.array(p.model.lens) + rng.integers(0, 30, R), 70 * 16)).tolist())
    p.compact()
    p.resize([70 * 16] * R)               # more than there are


def test_steps_captured_in_a_graph():
    say("pages graph")
    p = Pair(8, 6, 40)
    want, parent = p.ints([-1] * 8), p.ints([-1] * 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.pages.fork(parent)
        p.pages.resize(want)
    p.check()
    rng = np.random.default_rng(5)
    for i in range(6):
        w = np.minimum(np.array(p.model.lens) + rng.integers(0, 9, 8), 96).tolist()
        f = np.where(rng.random(8) < 0.3, rng.integers(0, 8, 8), -1).tolist()
        p.model.fork(f)
        for a, b, n in p.model.resize(w):
            for t in (p.k, p.v):
                t[:, b, :, :n] = t[:, a, :, :n]
        want.copy_(p.ints(w))
        parent.copy_(p.ints(f))
        graph.replay()
        torch.cuda.synchronize()
        p.check(f"replay {i}")
        if i == 3:
            p.compact()


def test_two_graphs_and_eager_calls_share_the_tables():
    say("pages two graphs")
    p = Pair(6, 5, 24)
    want, parent = p.ints([-1] * 6), p.ints([-1] * 6)
    grow, spread = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(grow):
        p.pages.resize(want)
    with torch.cuda.graph(spread):
        p.pages.fork(parent)
        p.pages.resize(want)
        p.pages.compact()
    rng = np.random.default_rng(11)
    for i in range(5):
        w = np.minimum(np.array(p.model.lens) + rng.integers(0, 20, 6), 80).tolist()
        for a, b, n in p.model.resize(w):
            for t in (p.k, p.v):
                t[:, b, :, :n] = t[:, a, :, :n]
        want.copy_(p.ints(w))
        grow.replay()
        p.check(f"grow {i}")
        f = np.where(rng.random(6) < 0.4, rng.integers(0, 6, 6), -1).tolist()
        p.model.fork(f)
        w = [max(n - int(rng.integers(0, 5)), 0) if rng.random() < 0.5 else min(n + 1, 80) for n in p.model.lens]
        for a, b, n in p.model.resize(w):
            for t in (p.k, p.v):
                t[:, b, :, :n] = t[:, a, :, :n]
        moves = p.model.compact()
        for t in (p.k, p.v):
            old = t.clone()
            for a, b in moves:
                t[:, b] = old[:, a]
        parent.copy_(p.ints(f))
        want.copy_(p.ints(w))
        spread.replay()
        p.check(f"spread {i}")
        p.resize([0 if r == i else n for r, n in enumerate(p.model.lens)])


def test_keys_follow_their_request():
    """Tables as a decode step uses them: two answers forked from one prompt write different tokens and each attends to its own."""
    say("pages and attention")
    H, D, P = 4, 64, 16
    cache = mlora.KVCache(1, 12, H, D, page_tokens=P)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    pages = mlora.KVPages(cache, 3, 4)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((25, H, D), device="cuda", generator=g).half() for _ in range(2))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")        # noqa: E731
    pages.resize(ints([20, 0, 0]))
    mlora.kv_append(None, k[:20], v[:20], cache, 0, mlora.KVBatch(ints([0] * 20), ints(list(range(20))), pages.table), None)
    pages.fork(ints([-1, 0, -1]))
    pages.resize(ints([21, 21, -1]))
    batch = mlora.KVBatch(ints([0, 1]), ints([20, 20]), pages.table)
    mlora.kv_append(None, k[20:22], v[20:22], cache, 0, batch, None)
    q = torch.randn((2, H, D), device="cuda", generator=g).half()
    out = mlora.prefix_attention(q, cache, 0, mlora.plan_attention(batch, cache, H))
    for r in range(2):
        kk, vv = (torch.cat((t[:20], t[20 + r:21 + r])).cpu().double() for t in (k, v))
        for h in range(H):
            s = kk[:, h] @ q[r, h].cpu().double() / 8
            want = torch.softmax(s, 0) @ vv[:, h]
            # weights and result in fp16, scores and sums in fp32: three half steps of fp16 of values up to the largest
            assert (out[r, h].cpu().double() - want).abs().max() <= 4 * 2.0 ** -11 * vv[:, h].abs().max()
