"""The largest batches, tables and numbers of heads that the attention takes, and inputs among the types' smallest values."""
import numpy as np
import pytest
import torch

import mlora
from gpu_common import say
from step_ref import attention_exact, check, f64, store_bound, w4_exact
from test_gpu_w4 import weight

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def i32(a):
    return torch.as_tensor(a, dtype=torch.int32).cuda()


def keys(cache, head, spans):
    """Rows of the given (page, number) spans."""
    return [np.concatenate([f64(t[0, p, head, :n]) for p, n in spans]) for t in (cache.k, cache.v)]


@pytest.mark.parametrize("heads, kv", [(1024, 1024), (1024, 1), (32, 8)])
def test_8192_tokens_behind_4096_prefixes(heads, kv):
    say(f"attention 8192 tokens, 4096 prefixes, {heads}/{kv} heads")
    T, F, P, D = 8192, 4096, 16, 64
    cache = mlora.KVCache(1, 300, kv, D, page_tokens=P, dtype=BF16)
    cache.k.normal_()
    cache.v.normal_()
    rng = np.random.default_rng(heads + kv)
    ppages, pages = rng.integers(0, 300, (F, 2)), rng.integers(0, 300, (T, 1))
    plen, own, of = rng.integers(1, 2 * P + 1, F), rng.integers(1, P + 1, T), rng.integers(-1, F, T)
    pos = own - 1 + np.where(of >= 0, plen[of], 0)
    batch = mlora.KVBatch(i32(range(T)), i32(pos), i32(pages), i32(of), i32(ppages), i32(plen))
    q = torch.randn((T, heads, D), device="cuda").to(BF16)
    out = mlora.prefix_attention(q, cache, 0, mlora.plan_attention(batch, cache, heads))
    for t in list(rng.integers(0, T, 12)) + [0, T - 1]:
        for h in (0, heads // 2 + 1, heads - 1):
            f, spans = of[t], []
            if f >= 0:
                spans = [(ppages[f, i], min(P, plen[f] - P * i)) for i in range(2) if plen[f] > P * i]
            k, v = keys(cache, h // (heads // kv), spans + [(pages[t, 0], own[t])])
            want, bound = attention_exact(f64(q[t, h]), k, v, D ** -0.5, BF16)
            check(out[t, h], want, bound, f"token {t} head {h}")


@pytest.mark.parametrize("there", [[0], [4194303], [7, 2000000, 4194302]])
def test_a_table_of_2_to_the_30_keys(there):
    """Keys on a few of 2^22 pages: the others are absent."""
    say(f"attention table of 2^30 keys, pages {there}")
    n, P = 1 << 22, 256
    cache = mlora.KVCache(1, 4, 2, 64, page_tokens=P, dtype=F16)
    cache.k.normal_()
    cache.v.normal_()
    pages = torch.full((2, n), -1, dtype=torch.int32, device="cuda")
    for i, p in enumerate(there):
        pages[1, p] = i + 1
    batch = mlora.KVBatch(i32([1, 0]), i32([n * P - 1, n * P - 5]), pages)
    q = torch.randn((2, 4, 64), device="cuda").to(F16)
    out = mlora.prefix_attention(q, cache, 0, mlora.plan_attention(batch, cache, 4))
    assert (out[1] == 0).all()
    for h in range(4):
        k, v = keys(cache, h // 2, [(i + 1, P) for i in range(len(there))])
        want, bound = attention_exact(f64(q[0, h]), k, v, 64 ** -0.5, F16)
        check(out[0, h], want, bound, f"head {h}")


@pytest.mark.parametrize("T", [3, 40])
def test_subnormal_values(T):
    """fp16 values below 2^-14 count in products of 4-bit weights, and as queries, keys and values."""
    say(f"subnormal fp16 T={T}")
    codes, scales, z = weight(520, 72, 64, True, F16, 2)
    x = (torch.randn((T, 520), device="cuda") * 2.0 ** -18).to(F16)
    y = torch.empty((T, 72), device="cuda", dtype=F16)
    scales = (scales.float() * 256).to(F16)
    mlora.w4_gemv([y], [x], [mlora.W4Weight(codes, scales, z, group=64)])
    want, bound = w4_exact(x, codes, scales, z, 64)
    check(y, want, bound + store_bound(np.abs(want) + bound, F16))
    cache = mlora.KVCache(1, 6, 1, 64, dtype=F16)
    cache.k.copy_(torch.randn(cache.k.shape) * 2.0 ** -18)
    cache.v.copy_(torch.randn(cache.v.shape) * 2.0 ** -18)
    batch = mlora.KVBatch(i32(range(T)), i32([69] * T), i32([[3, 1, 4, 0, 5]] * T))
    q = (torch.randn((T, 1, 64), device="cuda") * 2.0 ** -17).to(F16)
    out = mlora.prefix_attention(q, cache, 0, mlora.plan_attention(batch, cache, 1), scale=2.0 ** 34)
    k, v = keys(cache, 0, [(3, 16), (1, 16), (4, 16), (0, 16), (5, 6)])
    for t in range(T):
        want, bound = attention_exact(f64(q[t, 0]), k, v, 2.0 ** 34, F16)
        check(out[t, 0], want, bound, f"token {t}")
