"""Rotation and append to the paged cache against the 64-bit rotation; the cache's other rows stay as they were, bit for bit."""
import numpy as np
import pytest
import torch

import mlora
from gpu_common import say
from step_ref import check, f64, rope_exact, store_bound

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def run(T, n_req, heads, kv, D, P, rot, inter, dtype, seed=0, prefix=0, in_place=False, with_q=True, fused=True, layers=2, pad=()):
    say(f"append T={T} req={n_req} heads={heads}/{kv} D={D} P={P} rot={rot} inter={inter} {dtype} prefix={prefix}")
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    max_pages = 6
    n_pages = n_req * max_pages + 3
    pages = rng.permutation(n_pages)[:n_req * max_pages].reshape(n_req, max_pages).astype(np.int32)
    places = rng.permutation(n_req * max_pages * P)[:T]
    req, own = places // (max_pages * P), places % (max_pages * P)
    of = rng.integers(-1, 1, n_req).astype(np.int32) if prefix else np.full(n_req, -1, np.int32)
    pos = own + np.where(of[req] >= 0, prefix, 0)
    req = req.astype(np.int32)
    req[list(pad)] = -1
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()     # noqa: E731
    batch = mlora.KVBatch(i32(req), i32(pos), i32(pages), i32(of) if prefix else None, None, i32([prefix]) if prefix else None)
    cache = mlora.KVCache(layers, n_pages, kv, D, page_tokens=P, dtype=dtype)
    for t in (cache.k, cache.v):
        t.copy_(torch.randn(t.shape, generator=g).to(dtype))
    before = [cache.k.clone(), cache.v.clone()]
    qkv = torch.randn((T, heads + 2 * kv, D), generator=g).to(dtype)
    dev = qkv.cuda()
    q, k, v = dev[:, :heads], dev[:, heads:heads + kv], dev[:, heads + kv:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    rope = mlora.RopeTable(int(pos.max()) + 1, rot, interleaved=inter) if rot else None
    out = None if in_place or not with_q else torch.full((T, heads, D), 3.0, dtype=dtype, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = mlora.kv_append(q if with_q else None, k, v, cache, 1, batch, rope, q_out=out, bad=bad)
    assert int(bad) == 0
    live = req >= 0
    if with_q:
        want, bound = rope_exact(qkv[:, :heads], pos, rot, inter)
        check(got[live], want[live], (bound + store_bound(np.abs(want) + bound, dtype))[live], "q")
        assert torch.equal(got[~torch.from_numpy(live)].cpu(), qkv[:, :heads][~live] if in_place else torch.full_like(qkv[:, :heads], 3.0)[~live])
    else:
        assert got is None
    want_k, bound_k = rope_exact(qkv[:, heads:heads + kv], pos, rot, inter)
    keep = torch.ones(cache.k[1].shape[:1] + (P,), dtype=torch.bool)
    for t in range(T):
        if req[t] < 0:
            continue
        page, row = int(pages[req[t], own[t] // P]), int(own[t] % P)
        keep[page, row] = False
        check(cache.k[1, page, :, row], want_k[t], bound_k[t] + store_bound(np.abs(want_k[t]) + bound_k[t], dtype), f"k of token {t}")
        assert torch.equal(cache.v[1, page, :, row].cpu(), qkv[t, heads + kv:])
    for now, was in zip((cache.k, cache.v), before):
        assert torch.equal(now[0], was[0])
        same = now[1].permute(0, 2, 1, 3).cpu()[keep]
        assert torch.equal(same, was[1].permute(0, 2, 1, 3).cpu()[keep])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T, heads, kv, D, P, rot", [(1, 8, 8, 128, 16, 128), (7, 8, 2, 128, 32, 64), (20, 5, 1, 64, 16, 64),
                                                     (33, 12, 4, 64, 256, 16), (3, 64, 8, 128, 64, 128)])
def test_append(T, heads, kv, D, P, rot, inter, dtype):
    run(T, max(2, T // 2), heads, kv, D, P, rot, inter, dtype, seed=T)


def test_without_rotation_q_and_with_plain_rows():
    run(9, 4, 4, 2, 64, 16, 0, False, F16)
    run(9, 4, 4, 2, 64, 16, 32, True, F16, with_q=False)
    run(9, 4, 4, 2, 128, 16, 128, False, BF16, fused=False)


def test_in_place():
    run(17, 5, 8, 2, 128, 16, 128, False, BF16, in_place=True, pad=(0, 9, 16))
    run(17, 5, 8, 2, 64, 16, 32, True, F16, in_place=True)


def test_many_tokens():
    run(3000, 40, 4, 2, 128, 16, 128, False, F16, seed=3, layers=2)


def test_rows_without_a_request_stay():
    run(12, 5, 4, 4, 128, 16, 128, False, F16, pad=(0, 5, 6, 11))


@pytest.mark.parametrize("prefix", [1, 17, 100003])
def test_behind_a_prefix_at_far_positions(prefix):
    run(25, 6, 4, 2, 128, 16, 128, False, F16, prefix=prefix, seed=prefix)


def test_tokens_that_no_table_holds_are_left_out_and_counted():
    P, n_pages, D = 16, 8, 64
    cache = mlora.KVCache(1, n_pages, 2, D, page_tokens=P, dtype=F16)
    cache.k.fill_(1.0)
    cache.v.fill_(1.0)
    pages = torch.tensor([[0, 1], [2, -1], [3, n_pages], [4, 5]], dtype=torch.int32, device="cuda")
    #      good  pages' end  page -1  page n_pages  request 4  position -1  before its prefix  beyond the table  padding  good (behind its prefix)
    req = [0, 0, 1, 2, 4, 0, 3, 0, -1, 3]
    pos = [3, 32, 20, 17, 0, -1, 9, 40, 5, 10]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")     # noqa: E731
    batch = mlora.KVBatch(i32(req), i32(pos), pages, i32([-1, -7, 1, 0]), None, i32([10]))
    rope = mlora.RopeTable(40, D)
    x = torch.randn((10, 2, D), device="cuda").to(F16)
    out = torch.full((10, 2, D), 2.0, device="cuda", dtype=F16)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    mlora.kv_append(x, x, x, cache, 0, batch, rope, q_out=out, bad=bad)
    assert int(bad) == 7
    written = torch.zeros((n_pages, P), dtype=torch.bool)
    written[0, 3] = written[4, 0] = True
    assert ((cache.v[0] == 1.0).all(-1).all(1).cpu() == ~written).all()
    assert torch.equal(cache.v[0, 0, :, 3], x[0]) and torch.equal(cache.v[0, 4, :, 0], x[9])
    untouched = [t for t in range(10) if t not in (0, 9)]
    assert (out[untouched] == 2.0).all()
    mlora.kv_append(x, x, x, cache, 0, batch, rope, q_out=out)               # not counted
    assert int(bad) == 7


def test_offsets_past_32_bits():
    """A layer's slab of more than 2^32 elements, its last page."""
    n_pages = (1 << 32) // (8 * 256 * 128) + 3
    cache = mlora.KVCache(1, n_pages, 8, 128, page_tokens=256, dtype=F16)
    x = torch.randn((2, 8, 128), device="cuda").to(F16)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")     # noqa: E731
    cache.v[:, 0].zero_()
    batch = mlora.KVBatch(i32([0, 0]), i32([255, 256]), i32([[0, n_pages - 1]]))
    mlora.kv_append(None, x, x, cache, 0, batch, None)
    assert torch.equal(cache.k[0, 0, :, 255], x[0]) and torch.equal(cache.k[0, n_pages - 1, :, 0], x[1])
    assert torch.equal(cache.v[0, n_pages - 1, :, 0], x[1]) and not cache.v[0, 0, :, :255].any()


def test_captured_call_replays():
    cache = mlora.KVCache(1, 8, 2, 64, dtype=F16)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")     # noqa: E731
    batch = mlora.KVBatch(i32([0, 1]), i32([0, 0]), i32([[0, 1], [2, 3]]))
    rope = mlora.RopeTable(64, 64)
    x = torch.randn((2, 2, 64), device="cuda").to(F16)
    out = torch.empty_like(x)
    mlora.kv_append(x, x, x, cache, 0, batch, rope, q_out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mlora.kv_append(x, x, x, cache, 0, batch, rope, q_out=out)
    for i in range(4):
        batch.tok_pos.fill_(5 * i)
        x.copy_(torch.randn((2, 2, 64), device="cuda").to(F16))
        graph.replay()
        torch.cuda.synchronize()
        want, bound = rope_exact(x, [5 * i] * 2, 64, False)
        bound = bound + store_bound(np.abs(want) + bound, F16)
        check(out, want, bound, f"replay {i}")
        for t, first in enumerate((0, 2)):
            check(cache.k[0, first + 5 * i // 16, :, 5 * i % 16], want[t], bound[t])
    assert f64(cache.v).shape == (1, 8, 2, 16, 64)
