"""Rows whose result is made of small softmax weights, keys whose scores are infinite, and scales at the ends of their range."""
import numpy as np
import pytest
import torch

import mlora
from gpu_common import say
from step_ref import HALF, TINY, U32, Scene, check, f64, store_bound

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
INF = float("inf")


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


class Scores:
    """A cache whose first n keys have given scores with any q whose first element is one (the others meet zeros), and requests that all
    read these keys: `own` of them as their own, `behind` as a prefix.  With as many own readers as ranges fill the device every list is one
    range, so a wavefront meets long stretches."""

    def __init__(self, scores, heads, kv, D, dtype, own, behind, seed=0):
        n, P = len(scores), 64
        g = torch.Generator().manual_seed(seed)
        self.n, self.D, self.heads, self.kv = n, D, heads, kv
        n_pages = -(-n // P)
        self.cache = mlora.KVCache(1, n_pages + 1, kv, D, page_tokens=P, dtype=dtype)
        k = torch.zeros((n_pages + 1, P, D))
        k[:n_pages].view(-1, D)[:n, 0] = torch.as_tensor(scores, dtype=torch.float32)
        self.cache.k.copy_(k[None, :, None].expand(1, -1, kv, -1, -1))
        self.scores = f64(k.to(dtype)[:n_pages].reshape(-1, D)[:n, 0])
        self.v = (torch.rand((n_pages + 1, kv, P, D), generator=g) + 0.5).to(dtype)
        self.cache.v.copy_(self.v[None])
        T = own + behind
        # a request behind the prefix has no key of its own yet
        pages = [list(range(n_pages))] * own + [[n_pages] + [-1] * (n_pages - 1)] * behind
        self.batch = mlora.KVBatch(i32(range(T)), i32([n - 1] * own + [n - 1] * behind), i32(pages),
                                   i32([-1] * own + [0] * behind) if behind else None, i32([list(range(n_pages))]) if behind else None,
                                   i32([n]) if behind else None)
        q = torch.randn((T, heads, D), generator=g)
        q[:, :, 0] = 1.0
        self.q = q.to(dtype).cuda()
        self.T = T

    def values(self, head):
        return f64(self.v[:-1, head * self.kv // self.heads].reshape(-1, self.D)[:self.n])

    def run(self, scale=1.0):
        plan = mlora.plan_attention(self.batch, self.cache, self.heads)
        return mlora.prefix_attention(self.q, self.cache, 0, plan, scale=scale)


# one row of own keys and streaming loads, two tiles of own rows, 3 and 40 rows behind a prefix, 70 that share the rows instead
LAYOUTS = [(8, 8, 64, 0), (256, 8, 64, 0), (8, 8, 64, 3), (8, 8, 64, 40), (8, 8, 64, 70)]      # heads, key heads, own, behind


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads, kv, own, behind", LAYOUTS)
def test_many_small_weights(heads, kv, own, behind, D):
    """Keys 16 below a few that have all but the last thousandth of the weight, and zeros as these few's values: what the result is made of are
    the small weights.  In fp16 e^-16.2 is one and a half of the smallest steps above nothing."""
    say(f"attention small weights heads {heads}/{kv} own {own} behind {behind} D={D}")
    n = 8192
    rng = np.random.default_rng(D + behind)
    scores = -16.0 - rng.integers(8, 24, n) / 64.0
    s = Scores(scores, heads, kv, D, F16, own, behind)
    # a dominant key in each eighth of the list: in every wavefront's share, or in every other one's
    top = [q * (n // 8) + 5 for q in range(8)]
    for t in top:
        s.cache.k[0, t // 64, :, t % 64, 0] = 0.0
        s.cache.v[0, t // 64, :, t % 64] = 0.0
        s.v[t // 64, :, t % 64] = 0.0
        s.scores[t] = 0.0
    out = s.run()
    p = np.exp(s.scores)
    l = p.sum()
    for t in (0, own - 1, own, s.T - 1):
        for h in (0, heads - 1):
            if t >= s.T:
                continue
            v = s.values(h)
            want = p @ v / l
            # A score is one product and its scaling: (2 + 6) U32 of 16.5 in the exponent; the exponential 2 steps; a weight's rounding half a step of
            # fp16 relative, or half of its smallest step where the largest weight is 2^14; sums of n terms in fp32 in both, joined at the end
            rel = 2 * np.expm1(8 * U32 * 16.5 * 1.4427) + 2 * 2.0 ** -22 + 2 * HALF[F16] / (1 - HALF[F16]) + 2 * (n + 80) * U32
            bound = rel * want + 2 * n * TINY[F16] * 2.0 ** -14 * np.abs(v).max(0) / l
            check(out[t, h], want, bound + store_bound(want + bound, F16), f"token {t} head {h}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads, kv, own, behind", LAYOUTS + [(4, 2, 2, 0), (4, 2, 0, 6), (2, 1, 1, 80)])
def test_rows_whose_scores_are_all_minus_infinity(heads, kv, own, behind, dtype):
    """The softmax of nothing but minus infinities is NaN; one finite score among them has the whole weight, wherever it lies."""
    say(f"attention minus infinity heads {heads}/{kv} own {own} behind {behind} {dtype}")
    n = 700
    s = Scores(np.full(n, -INF), heads, kv, 64, dtype, own, behind)
    assert s.run().isnan().all()
    for at in (0, 333, n - 1):
        s.cache.k[0, at // 64, :, at % 64, 0] = 2.0
        out = s.run()
        for h in (0, heads - 1):
            want = torch.from_numpy(s.values(h)[at]).to(dtype).cuda()
            assert (out[:, h] == want).all()
        s.cache.k[0, at // 64, :, at % 64, 0] = -INF


def test_absent_keys_are_not_infinite_ones():
    """Every page missing: no key at all, and zeros.  One page there, and its scores minus infinity: NaN."""
    s = Scores(np.full(200, -INF), 4, 2, 64, F16, 2, 3)
    s.batch.pages.fill_(-1)
    s.batch.prefix_pages.fill_(-1)
    assert (s.run() == 0).all()
    s.batch.pages[1, 2] = 1
    out = s.run()
    assert out[1].isnan().all() and (out[0] == 0).all() and (out[2:] == 0).all()
    s.batch.prefix_pages[0, 3] = 0
    out = s.run()
    assert out[1:].isnan().all() and (out[0] == 0).all()


@pytest.mark.parametrize("n_req", [3, 70])
def test_scales_at_the_ends_of_their_range(n_req):
    """A scale of zero gives every key the same weight however far the scores are apart; one near the smallest float meets scores that make up for
    it; 2^127 leaves the largest score the whole weight."""
    say(f"attention scales {n_req}")
    s = Scene([(0, 9 + i) for i in range(n_req)], [150], 2, 1, 64, 16, BF16, seed=n_req)
    s.k = (s.k.double() * 2.0 ** 60).to(BF16)
    s.cache.k.copy_(s.k)
    s.q = (s.q.double() * 2.0 ** 55).to(BF16)
    s.dev_q = s.q.cuda()
    plan = mlora.plan_attention(s.batch, s.cache, 2)
    for scale in (0.0, 2.0 ** -118, -2.0 ** -118):
        s.compare(mlora.prefix_attention(s.dev_q, s.cache, 0, plan, scale=scale), scale=scale, what=f"scale {scale}")
    s.q, s.k = (s.q.double() * 2.0 ** -65).to(BF16), (s.k.double() * 2.0 ** -60).to(BF16)
    s.dev_q = s.q.cuda()
    s.cache.k.copy_(s.k)
    out = f64(mlora.prefix_attention(s.dev_q, s.cache, 0, plan, scale=2.0 ** 127))
    for t in range(n_req):
        k, v = (np.concatenate([s.rows(w, 0, s.prefix_lists[0], 150, 0), s.rows(w, 0, s.req_lists[t], 9 + t, 0)]) for w in "kv")
        for h in range(2):
            score = k @ f64(s.q[t, h])
            second, first = np.sort(score)[-2:]
            if first - second > 1e-4 * np.abs(score).max():      # or fp32 may not tell the two apart
                assert (out[t, h] == v[score.argmax()]).all()
