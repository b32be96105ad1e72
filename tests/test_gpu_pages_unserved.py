"""Rows that a resize could not serve: what the device says of them, and that a step which goes by it leaves other rows' keys as they were."""
import numpy as np
import pytest
import torch

import mlora
from test_gpu_pages import Pair
from test_gpu_token_step import build
from test_gpu_token_step_mx4 import weights_of

pytestmark = pytest.mark.gpu


def grown_by(p, want):
    before = list(p.model.lens)
    p.resize(want)
    return [r if n > m else -1 for r, (m, n) in enumerate(zip(before, p.model.lens))]


def test_rows_that_got_longer():
    p = Pair(6, 8, 7)
    assert p.pages.grown.tolist() == [-1] * 6
    assert grown_by(p, [16, 0, 20, 1, -1, 0]) == p.pages.grown.tolist() == [0, -1, 2, 3, -1, -1]
    assert grown_by(p, [16, 0, 19, 2, 200, 17]) == p.pages.grown.tolist() == [-1, -1, -1, 3, -1, 5]        # row 4: more than max_pages
    assert grown_by(p, [16, 17, 19, 2, -1, 18]) == p.pages.grown.tolist() == [-1, -1, -1, -1, -1, 5]       # row 1: two pages, one is free
    assert p.model.failed == 2
    p.resize([17, -1, -1, -1, -1, -1])
    assert p.pages.grown.tolist() == [0, -1, -1, -1, -1, -1]
    p.compact()
    assert p.pages.grown.tolist() == [0, -1, -1, -1, -1, -1]
    p.fork([-1] * 6)
    assert p.pages.grown.tolist() == [-1] * 6
    p.resize([18, -1, -1, -1, -1, -1])
    p.pages.adopt(p.pages.table.clone(), p.pages.lens.clone())
    assert p.pages.grown.tolist() == [-1] * 6
    p.check()


# rows of one thread each or several, pages given back by the same launch or one of its own
@pytest.mark.parametrize("R, M", [(40, 8), (300, 300), (1500, 40), (1500, 70)])
def test_rows_that_got_longer_in_every_form(R, M):
    rng = np.random.default_rng(R + M)
    p = Pair(R, M, 3 * R, layers=1, kv_heads=1)
    p.resize(rng.integers(0, 60, R).tolist())
    p.fork(np.where(rng.random(R) < 0.5, rng.integers(0, R, R), -1).tolist())
    for _ in range(4):
        lens = np.array(p.model.lens)
        kind = rng.random(R)
        want = np.where(kind < 0.6, lens + rng.integers(1, 40, R), np.where(kind < 0.7, 0, np.where(kind < 0.8, np.maximum(lens - 3, 0), np.where(kind < 0.9, lens, -1))))
        assert grown_by(p, want.tolist()) == p.pages.grown.tolist()
    assert p.model.failed > 0


class Step:
    """Row 0's 20 tokens, two forks of it, and a row of 17 tokens; the cache's four pages are all in use."""

    def __init__(self):
        self.pool, _, self.cache, self.g = build(1, 128, 4, 2, 64, 3, torch.float16, 4, 1)
        _, packed = weights_of(1, self.pool.projections, torch.float16, 2)
        for t in (self.cache.k, self.cache.v):
            t.copy_(torch.randn(t.shape, device="cuda", generator=self.g))
        self.pages = mlora.KVPages(self.cache, 4, 3)
        self.pages.resize(self.ints([20, 0, 0, 17]))
        self.pages.fork(self.ints([-1, 0, 0, -1]))
        self.step = mlora.TokenStep(self.pool, self.cache, packed, 4, mlora.RopeTable(64, 64))
        self.want, self.pos, self.slots = self.ints([-1] * 4), self.ints([0] * 4), self.ints([0, 1, 2, -1])
        self.x = torch.randn((4, 128), device="cuda", generator=self.g).half()
        self.batch = mlora.KVBatch(self.pages.grown, self.pos, self.pages.table)

    @staticmethod
    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def once(self, positions="lens"):
        self.pages.resize(self.want)
        torch.sub(self.pages.lens if positions == "lens" else self.want, 1, out=self.pos)
        self.step.begin(self.batch, self.slots)
        return self.step.layer(0, self.x)

    def held(self, r, n):
        """Keys and values of a row's first n tokens."""
        page = self.pages.table[r].long().tolist()
        return [torch.cat([t[0, p] for p in page[:-(-n // 16)]], 1)[:, :n].clone() for t in (self.cache.k, self.cache.v)]


@pytest.mark.parametrize("positions", ["lens", "want"])
def test_a_step_without_room_leaves_shared_pages_alone(positions):
    print(f"[gpu-case] step without a free page, positions from {positions}", flush=True)
    s = Step()
    before = [s.held(r, n) for r, n in enumerate((20, 20, 20, 17))]
    k0, v0 = s.cache.k.clone(), s.cache.v.clone()
    s.want.copy_(s.ints([21, 21, 21, 18]))
    out = s.once(positions)
    torch.cuda.synchronize()
    assert s.pages.grown.tolist() == [-1, -1, -1, 3] and s.pages.lens.tolist() == [20, 20, 20, 18] and s.pages.failed.tolist() == [3] and int(s.step.bad) == 0
    assert not out[:3].any() and out[3].any()
    page = int(s.pages.table[3, 1])
    for t, t0 in ((s.cache.k, k0), (s.cache.v, v0)):
        assert not torch.equal(t[0, page, :, 1], t0[0, page, :, 1])         # the served row's token
        t0[0, page, :, 1] = t[0, page, :, 1]
        assert torch.equal(t, t0)                                           # and nothing else
    # with room for the copies, the rows go on from what they had
    s.want.copy_(s.ints([21, 21, 21, 0]))
    out = s.once(positions)
    torch.cuda.synchronize()
    assert s.pages.grown.tolist() == [0, 1, 2, -1] and s.pages.lens.tolist() == [21, 21, 21, 0] and int(s.step.bad) == 0
    assert out[:3].any() and not out[3].any()
    for r in range(3):
        assert all(torch.equal(a, b) for a, b in zip(s.held(r, 20), before[r])), r
    v = s.step.qkv[2].view(4, -1, 64)
    for r in range(3):
        assert torch.equal(s.held(r, 21)[1][:, 20], v[r])


def test_captured_steps_with_and_without_room():
    print("[gpu-case] captured step without a free page", flush=True)
    s = Step()
    start = s.pages.state.clone()
    s.once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.once()
    s.pages.state.copy_(start)
    for want, grown in (([21, 21, 21, 18], [-1, -1, -1, 3]), ([21, 21, 21, 19], [-1, -1, -1, 3]), ([21, 21, 21, 0], [0, 1, 2, -1]), ([22, 22, 22, 0], [0, 1, 2, -1]),
                        ([-1, 23, 0, 1], [-1, 1, -1, 3]), ([33, 24, 0, 2], [-1, 1, -1, 3])):
        s.want.copy_(s.ints(want))
        s.x.copy_(torch.randn((4, 128), device="cuda", generator=s.g))
        state, k0, v0 = s.pages.state.clone(), s.cache.k.clone(), s.cache.v.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert s.pages.grown.tolist() == grown, want
        for r in range(4):
            if grown[r] < 0:
                assert not out[r].any(), (want, r)
        got, after, k, v = out.clone(), s.pages.state.clone(), s.cache.k.clone(), s.cache.v.clone()
        s.pages.state.copy_(state)
        s.cache.k.copy_(k0)
        s.cache.v.copy_(v0)
        assert torch.equal(s.once(), got) and torch.equal(s.pages.state, after) and torch.equal(s.cache.k, k) and torch.equal(s.cache.v, v), want
