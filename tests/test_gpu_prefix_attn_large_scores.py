"""Scores beyond 2^24 that are no powers of two: the largest key of a row has the whole weight, and the row is its value."""
import numpy as np
import pytest
import torch

import mlora
from gpu_common import say
from step_ref import Scene, f64

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype, q_power, k_power, scale", [(F16, 11, 11, 4.0), (F16, 13, 13, 2.0 ** 20), (BF16, 14, 14, 1.0), (BF16, 50, 50, 0.3),
                                                            (BF16, 14, 14, -1.0)])
@pytest.mark.parametrize("n_req, heads", [(1, 2), (3, 2), (3, 20), (40, 1), (70, 1)])
def test_the_largest_score_has_the_whole_weight(n_req, heads, dtype, q_power, k_power, scale):
    say(f"attention scores of 2^{q_power + k_power} {dtype} scale {scale} requests {n_req} heads {heads}")
    for prefix in (0, 300):
        s = Scene([(0 if prefix else -1, 40 + 3 * i) for i in range(n_req)], [prefix] if prefix else [], heads, 1, 64, 16, dtype, seed=n_req + heads)
        s.k = (s.k.double().clamp(-3.5, 3.5) * 2.0 ** k_power).to(dtype)
        s.cache.k.copy_(s.k)
        s.q = (s.q.double().clamp(-3.5, 3.5) * 2.0 ** q_power).to(dtype)
        s.dev_q = s.q.cuda()
        plan = mlora.plan_attention(s.batch, s.cache, heads)
        out = f64(mlora.prefix_attention(s.dev_q, s.cache, 0, plan, scale=scale))
        alone = 0
        for t in range(n_req):
            parts = [[s.rows(w, 0, s.prefix_lists[0], prefix, 0)] if prefix else [] for w in "kv"]
            k, v = (np.concatenate(p + [s.rows(w, 0, s.req_lists[t], 40 + 3 * t, 0)]) for p, w in zip(parts, "kv"))
            for h in range(heads):
                score = k @ f64(s.q[t, h]) * scale
                second, first = np.sort(score)[-2:]
                # fp32 sums of 64 products: 66 roundings of the sum of magnitudes for each of the two
                if first - second > 2 * 66 * 2.0 ** -24 * (np.abs(k) @ np.abs(f64(s.q[t, h]))).max() * abs(scale) + 64:
                    alone += 1
                    assert (out[t, h] == v[score.argmax()]).all(), (prefix, t, h)
        assert alone >= n_req * heads * 0.9
