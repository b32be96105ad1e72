"""Batches of more workgroups than one launch takes."""
import numpy as np
import pytest
import torch

import mlora
from gpu_common import say
from step_ref import check, store_bound, w4_exact
from test_gpu_w4 import weight

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def test_append_of_more_tokens_than_a_launch_has_workgroups():
    T = (1 << 24) + 1003
    say(f"append T={T}")
    P, D = 256, 64
    pages = -(-T // P)
    cache = mlora.KVCache(1, pages, 1, D, page_tokens=P, dtype=F16)
    cache.v.zero_()
    i32 = dict(dtype=torch.int32, device="cuda")
    req = torch.zeros(T, **i32)
    req[5] = req[T - 2] = -1
    bad = torch.zeros(1, **i32)
    order = torch.randperm(pages, device="cuda").to(torch.int32)
    order[3] = pages                                                    # 256 tokens whose page is none
    batch = mlora.KVBatch(req, torch.arange(T, **i32), order[None])
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((T, 1, D), device="cuda", dtype=F16, generator=g) for _ in range(2))
    assert mlora.kv_append(None, k, v, cache, 0, batch, None, bad=bad) is None
    assert int(bad) == P
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[5] = keep[T - 2] = False
    keep[3 * P:4 * P] = False
    order[3] = 0
    for got, want in ((cache.k, k), (cache.v, v)):
        rows = got[0, order.long(), 0].view(-1, D)[:T]
        assert torch.equal(rows[keep], want[keep, 0])
    assert (cache.v[0, order.long(), 0].view(-1, D)[[5, T - 2]] == 0).all()


@pytest.mark.parametrize("group", [64, 128])
def test_product_of_more_blocks_than_a_launch_has_workgroups(group):
    T, hin, hout = (1 << 20) - 5, 8, 16456
    say(f"w4 T={T} {hin}->{hout} group={group}")
    codes, scales, z = weight(hin, hout, group, True, BF16, 1)
    w = mlora.W4Weight(codes, scales, z, group=group)
    x = torch.randn((T, hin), device="cuda").to(BF16)
    y = torch.full((T, hout), float("nan"), device="cuda", dtype=BF16)
    mlora.w4_gemv([y], [x], [w])
    for a in range(0, T, 1 << 16):
        assert torch.isfinite(y[a:a + (1 << 16)].sum(1, dtype=torch.float32)).all(), f"rows from {a}"
    rng = np.random.default_rng(1)
    rows = torch.from_numpy(np.sort(np.concatenate([rng.integers(0, T, 200), [0, T - 1], np.arange(1, T // 64, 997) * 64]))).cuda()
    want, bound = w4_exact(x[rows], codes, scales, z, group)
    check(y[rows], want, bound + store_bound(np.abs(want) + bound, BF16))
    before = y[rows].clone()
    mlora.w4_gemv([y], [x], [w], accumulate=True)
    check(y[rows], want + before.double().cpu().numpy(), bound + store_bound(np.abs(want) + bound + np.abs(before.double().cpu().numpy()), BF16))
