"""A decode step on microscaled weights over page tables on the device: prompts, answers forked from them, steps, one of them captured, a compaction."""
import numpy as np
import pytest
import torch

import mlora
import mx4_ref as ref
from pages_ref import Tables
from step_ref import HALF, TINY, U32, attention_exact, check, f64, rope_exact
from test_gpu_token_step import build, deltas

pytestmark = pytest.mark.gpu


def weights_of(L, widths, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    plain = [{n: (torch.randn(w, device="cuda", generator=g) * 0.05).to(dtype) for n, w in widths.items()} for _ in range(L)]
    return plain, [{n: mlora.MX4Weight.quantize(w) for n, w in layer.items()} for layer in plain]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads, kv, D", [(4, 2, 64), (4, 4, 128)])
def test_steps_of_forked_requests(heads, kv, D, dtype):
    print(f"[gpu-case] mx4 token step {heads}/{kv} D={D} {dtype}", flush=True)
    L, hin, N, R, P, M = 2, 264, 3, 5, 16, 6
    pool, _, cache, g = build(L, hin, heads, kv, D, N, dtype, 40, heads)
    plain, packed = weights_of(L, pool.projections, dtype, 1)
    pages = mlora.KVPages(cache, R, M)
    model = Tables([[] for _ in range(R)], [0] * R, range(40), 40, P, M)
    step = mlora.TokenStep(pool, cache, packed, heads, mlora.RopeTable(P * M, D))
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")          # noqa: E731
    slots = [0, -1, 2, 1, 0]

    def resize(want):
        model.resize(want)
        pages.resize(i32(want))
        assert pages.table.tolist() == model.table() and pages.lens.tolist() == model.lens

    def keys(layer, t, which, n):
        src = cache.k if which == "k" else cache.v
        return np.concatenate([f64(src[layer, p, :, :min(P, n - i * P)]) for i, p in enumerate(model.rows[t][:-(-n // P)])], 1)

    # prompts of 37 and 20 tokens, then three answers to the first and two to the second
    resize([37, 0, 0, 20, 0])
    for layer in range(L):
        n = 57
        k, v = (torch.randn((n, kv, D), device="cuda", generator=g).to(dtype) for _ in range(2))
        batch = mlora.KVBatch(i32([0] * 37 + [3] * 20), i32(list(range(37)) + list(range(20))), pages.table)
        mlora.kv_append(None, k, v, cache, layer, batch, None)
    model.fork([-1, 0, 0, -1, 3])
    pages.fork(i32([-1, 0, 0, -1, 3]))
    for turn in range(3):
        resize([n + 1 for n in model.lens])
        pos = [n - 1 for n in model.lens]
        batch = mlora.KVBatch(i32(range(R)), i32(pos), pages.table)
        step.begin(batch, i32(slots))
        for layer in range(L):
            x = torch.randn((R, hin), device="cuda", generator=g).to(dtype)
            before = {(t, w): keys(layer, t, w, pos[t]) for t in range(R) for w in "kv" if pos[t]}
            products = [torch.empty((R, w), dtype=dtype, device="cuda") for w in step.widths]
            mlora.mx4_gemm(products, [mlora.mx4_quantize(x)] * 3, [packed[layer][n] for n in "qkv"])
            xv = ref.values(*ref.quantize(f64(x)))
            wanted = []
            for y, name in zip(products, "qkv"):
                want, b = ref.gemm(xv, ref.values(*ref.quantize(f64(plain[layer][name].t()))))
                first = b + HALF[dtype] * (np.abs(want) + b) + TINY[dtype]
                check(y, want, first, f"base {name}")
                delta, mag = deltas(pool, layer, name, x, slots)
                bound = first + (hin + 80) * U32 * mag
                wanted.append((want + delta, bound + HALF[dtype] * (np.abs(want + delta) + bound) + TINY[dtype]))
            mlora.bgmv(products, [x] * 3, pool, layer, ["q", "k", "v"], i32(slots), plan=step.decode_plan)
            for y, (want, bound), name in zip(products, wanted, "qkv"):
                check(y, want, bound, name)
            out = step.layer(layer, x)
            torch.cuda.synchronize()
            assert int(step.bad) == 0
            q, k, v = (y.view(R, -1, D) for y in products)
            wk, bk = rope_exact(k, pos, D, False)
            for t in range(R):
                page, at = model.rows[t][pos[t] // P], pos[t] % P
                check(cache.k[layer, page, :, at], wk[t], bk[t] + HALF[dtype] * (np.abs(wk[t]) + bk[t]) + TINY[dtype], f"appended k {t}")
                assert torch.equal(cache.v[layer, page, :, at], v[t])
                for w in "kv":                        # nobody else's token got into what a request had
                    if pos[t]:
                        assert np.array_equal(keys(layer, t, w, pos[t]), before[t, w]), (turn, layer, t, w)
                for h in range(heads):
                    kk, vv = (keys(layer, t, w, pos[t] + 1)[h * kv // heads] for w in "kv")
                    want, bound = attention_exact(f64(step.qkv[0].view(R, heads, D)[t, h]), kk, vv, D ** -0.5, dtype)
                    check(out[t, h], want, bound, f"attention token {t} head {h}")
        if turn == 1:
            # one request ends, beams are reordered, and the pages in use move together
            resize([-1, -1, 0, -1, -1])
            model.fork([1, 0, 4, -1, -1])
            pages.fork(i32([1, 0, 4, -1, -1]))
            held = {(t, layer, w): keys(layer, t, w, model.lens[t]) for t in range(R) for layer in range(L) for w in "kv"}
            model.compact()
            pages.compact()
            assert pages.table.tolist() == model.table() and pages.live.tolist() == [sum(n > 0 for n in model.refs())]
            for (t, layer, w), was in held.items():
                assert np.array_equal(keys(layer, t, w, model.lens[t]), was)


def test_a_captured_step_replays():
    """Pages, plans, projections and attention in one graph; every replay against eager work on the same tables."""
    print("[gpu-case] mx4 token step graph", flush=True)
    pool, _, cache, g = build(1, 128, 4, 2, 64, 3, torch.float16, 40, 1)
    _, packed = weights_of(1, pool.projections, torch.float16, 2)
    pages = mlora.KVPages(cache, 6, 4)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")          # noqa: E731
    pages.resize(i32([30, 0, 3, 17, 0, 44]))
    pages.fork(i32([-1, 0, -1, -1, 3, -1]))
    step = mlora.TokenStep(pool, cache, packed, 4, mlora.RopeTable(64, 64))
    slots, want, pos, x = i32([0, 1, 2, -1, 0, 0]), i32([-1] * 6), i32([0] * 6), torch.randn((6, 128), device="cuda", generator=g).half()
    batch = mlora.KVBatch(i32(range(6)), pos, pages.table)

    def once():
        pages.resize(want)
        torch.sub(pages.lens, 1, out=pos)
        step.begin(batch, slots)
        return step.layer(0, x)
    once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for i in range(4):
        want.copy_(pages.lens + 1)
        x.copy_(torch.randn((6, 128), device="cuda", generator=g))
        start, k0, v0 = pages.state.clone(), cache.k.clone(), cache.v.clone()
        graph.replay()
        torch.cuda.synchronize()
        got, state, k = out.clone(), pages.state.clone(), cache.k.clone()
        pages.state.copy_(start)
        cache.k.copy_(k0)
        cache.v.copy_(v0)
        assert torch.equal(once(), got) and torch.equal(pages.state, state) and torch.equal(cache.k, k), i


def test_batches_of_no_and_of_few_tokens_in_turn():
    """One step object over batches whose operands share a buffer, one of them empty."""
    print("[gpu-case] mx4 token step batches in turn", flush=True)
    pool, _, cache, g = build(1, 136, 4, 2, 64, 3, torch.float16, 40, 1)
    _, packed = weights_of(1, pool.projections, torch.float16, 2)
    step = mlora.TokenStep(pool, cache, packed, 4, mlora.RopeTable(64, 64))
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")          # noqa: E731
    for T in (5, 0, 8, 0, 6, 1, 33):
        batch = mlora.KVBatch(i32(range(T)), i32([0] * T), i32([[t] for t in range(max(T, 1))]))
        x = torch.randn((T, 136), device="cuda", generator=g).half()
        step.begin(batch, i32([-1] * T))
        assert step.layer(0, x).shape[0] == T
        v = torch.empty((T, step.widths[2]), dtype=torch.float16, device="cuda")
        mlora.mx4_gemm([v], [mlora.mx4_quantize(x)], [packed[0]["v"]])
        assert torch.equal(step.qkv[2], v), T


def test_kinds_of_weights():
    pool, _, cache, g = build(1, 128, 4, 2, 64, 3, torch.float16, 8, 1)
    plain, packed = weights_of(1, pool.projections, torch.float16, 2)
    mixed = dict(packed[0], q=mlora.W4Weight.quantize(plain[0]["q"], 32))
    with pytest.raises(ValueError):
        mlora.TokenStep(pool, cache, [mixed], 4)
    with pytest.raises(ValueError):
        mlora.TokenStep(pool, cache, [dict(packed[0], q=packed[0]["k"])], 4)
    # layers of either kind
    pool, _, cache, g = build(2, 128, 4, 2, 64, 3, torch.float16, 8, 1)
    plain, packed = weights_of(2, pool.projections, torch.float16, 2)
    four = {n: mlora.W4Weight.quantize(w, 32) for n, w in plain[1].items()}
    step = mlora.TokenStep(pool, cache, [packed[0], four], 4, mlora.RopeTable(64, 64))
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")          # noqa: E731
    batch = mlora.KVBatch(i32([0, 1, -1]), i32([0, 0, 0]), i32([[0], [1], [2]]))
    x = torch.randn((3, 128), device="cuda", generator=g).half()
    step.begin(batch, i32([-1, -1, -1]))
    for layer in range(2):
        step.layer(layer, x)
        want = [torch.empty((3, w), dtype=torch.float16, device="cuda") for w in step.widths]
        if layer == 0:
            mlora.mx4_gemm(want, [mlora.mx4_quantize(x)] * 3, [packed[0][n] for n in "qkv"])
        else:
            mlora.w4_gemv(want, [x] * 3, [four[n] for n in "qkv"])
        assert torch.equal(step.qkv[2], want[2])                               # v: neither rotated nor changed by an adapter
