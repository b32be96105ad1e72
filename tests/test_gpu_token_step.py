"""The operators of a decode step together: 4-bit base projections, LoRA deltas, rotation and append, shared-prefix attention."""
import numpy as np
import pytest
import torch

import mlora
from mlora import trace_driver as td
from step_ref import HALF, TINY, U32, attention_exact, check, f64, rope_exact, w4_exact

pytestmark = pytest.mark.gpu


def build(L, hin, heads, kv, D, N, dtype, n_pages, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    widths = {"q": (hin, heads * D), "k": (hin, kv * D), "v": (hin, kv * D)}
    pool = mlora.AdapterPool(L, widths, N, N * 2, page_rows=8, max_rank=16, dtype=dtype)
    for slot in range(N):
        pool.allocate(slot, 8 if slot % 2 else 16, 0.5 + slot / 8)
    for rows in list(pool.a_rows.values()) + list(pool.b_rows.values()):
        rows.copy_(torch.randn(rows.shape, device="cuda", generator=g) * 0.05)
    weights = [{n: mlora.w4_quantize((torch.randn(w, device="cuda", generator=g) * 0.05).to(dtype), 32, symmetric=n == "q")
                for n, w in widths.items()} for _ in range(L)]
    cache = mlora.KVCache(L, n_pages, kv, D, dtype=dtype)
    cache.k.copy_(torch.randn(cache.k.shape, device="cuda", generator=g))
    cache.v.copy_(torch.randn(cache.v.shape, device="cuda", generator=g))
    return pool, weights, cache, g


def deltas(pool, layer, name, x, slots):
    """64-bit LoRA deltas, and a bound on the kernel's: fp32 sums over hin and the rank, the intermediate in fp32."""
    out, mag = [], []
    for t, s in enumerate(slots):
        if s < 0:
            out.append(np.zeros(pool.projections[name][1]))
            mag.append(out[-1])
            continue
        rows = pool.rows_of(s)
        a, b = f64(pool.a_rows[name][layer][rows]), f64(pool.b_rows[name][layer][rows])
        out.append(float(pool.h_scaling[s]) * (a @ f64(x)[t]) @ b)
        mag.append(float(pool.h_scaling[s]) * (np.abs(a) @ np.abs(f64(x)[t])) @ np.abs(b))
    return np.stack(out), np.stack(mag)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T, heads, kv, D", [(1, 4, 2, 64), (9, 8, 2, 64), (40, 4, 4, 128)])
def test_a_decode_step(T, heads, kv, D, dtype):
    """Each operator against 64 bits on what the one before it left: q, k, v as projected, as rotated and appended, and the attention over
    the cache as it then is."""
    print(f"[gpu-case] token step T={T} {heads}/{kv} D={D} {dtype}", flush=True)
    L, hin, N, prefix, own = 2, 256, 5, 50, 20
    pool, weights, cache, g = build(L, hin, heads, kv, D, N, dtype, 4 + 2 * T + 6, T)
    prompts = [cache.allocate(4), ]
    lists = [cache.allocate(2) for _ in range(T)]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")      # noqa: E731
    of = [0 if t % 3 else -1 for t in range(T)]
    lens = [1 + (7 * t) % own for t in range(T)]
    pos = [(prefix if f >= 0 else 0) + n - 1 for f, n in zip(of, lens)]
    slots = [t % (N + 1) - 1 for t in range(T)]
    batch = mlora.KVBatch(i32(range(T)), i32(pos), i32(lists), i32(of), i32(prompts), i32([prefix]))
    packed = [{n: mlora.W4Weight(*w, group=32) for n, w in layer.items()} for layer in weights]
    step = mlora.TokenStep(pool, cache, packed, heads, mlora.RopeTable(128, D))
    for again in range(2):                                                 # the second time from kept plans and buffers
        step.begin(batch, i32(slots))
        for layer in range(L):
            x = torch.randn((T, hin), device="cuda", generator=g).to(dtype)
            plain = [torch.empty((T, w), dtype=dtype, device="cuda") for w in step.widths]
            mlora.w4_gemv(plain, [x] * 3, [packed[layer][n] for n in "qkv"])
            mlora.bgmv(plain, [x] * 3, pool, layer, ["q", "k", "v"], i32(slots), plan=step.decode_plan)
            out = step.layer(layer, x)
            torch.cuda.synchronize()
            for y, name in zip(plain, "qkv"):
                want, b = w4_exact(x, *weights[layer][name], 32)
                delta, mag = deltas(pool, layer, name, x, slots)
                # the base product rounded, the sum with the delta rounded; the delta's own fp32 sums over hin and rank
                first = b + HALF[dtype] * (np.abs(want) + b) + TINY[dtype]
                bound = first + (hin + 80) * U32 * mag
                check(y, want + delta, bound + HALF[dtype] * (np.abs(want + delta) + bound) + TINY[dtype], f"{name} layer {layer}")
            q, k, v = (y.view(T, -1, D) for y in plain)
            wq, bq = rope_exact(q, pos, D, False)
            wk, bk = rope_exact(k, pos, D, False)
            check(step.qkv[0].view(T, heads, D), wq, bq + HALF[dtype] * (np.abs(wq) + bq) + TINY[dtype], "rotated q")
            for t in range(T):
                at = (lists[t][(lens[t] - 1) // 16], (lens[t] - 1) % 16)
                check(cache.k[layer, at[0], :, at[1]], wk[t], bk[t] + HALF[dtype] * (np.abs(wk[t]) + bk[t]) + TINY[dtype], f"appended k {t}")
                assert torch.equal(cache.v[layer, at[0], :, at[1]], v[t])
                pages = ([(p, 16) for p in prompts[0][:3]] + [(prompts[0][3], 2)] if of[t] >= 0 else []) + \
                        [(lists[t][0], min(16, lens[t]))] + ([(lists[t][1], lens[t] - 16)] if lens[t] > 16 else [])
                for h in range(heads):
                    kk, vv = (np.concatenate([f64(c[layer, p, h * kv // heads, :n]) for p, n in pages]) for c in (cache.k, cache.v))
                    want, bound = attention_exact(f64(step.qkv[0].view(T, heads, D)[t, h]), kk, vv, D ** -0.5, dtype)
                    check(out[t, h], want, bound, f"attention token {t} head {h}")


def test_a_captured_step_replays():
    pool, weights, cache, g = build(1, 128, 4, 2, 64, 3, torch.float16, 40, 1)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")      # noqa: E731
    T = 6
    lists = [cache.allocate(2) for _ in range(T)]
    prompt = cache.allocate(3)
    batch = mlora.KVBatch(i32(range(T)), i32([40] * T), i32(lists), i32([0] * T), i32([prompt]), i32([40]))
    slots = i32([0, 1, 2, -1, 0, 0])
    step = mlora.TokenStep(pool, cache, [{n: mlora.W4Weight(*w, group=32) for n, w in weights[0].items()}], 4, mlora.RopeTable(128, 64))
    x = torch.randn((T, 128), device="cuda", generator=g).half()

    def once():
        step.begin(batch, slots)
        return step.layer(0, x)
    once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for i in range(4):
        batch.tok_pos.copy_(i32([40 + i + t for t in range(T)]))
        x.copy_(torch.randn((T, 128), device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got, k = out.clone(), cache.k.clone()
        assert torch.equal(once(), got) and torch.equal(cache.k, k)


def test_buffers_do_not_add_up_over_batch_sizes():
    """Steps of every size to 33, up and down, keep a buffer for a power of two each; results are those of a step of its own."""
    pool, weights, cache, g = build(1, 128, 4, 2, 64, 3, torch.float16, 40, 1)
    ws = [{n: mlora.W4Weight(*w, group=32) for n, w in layer.items()} for layer in weights]
    rope = mlora.RopeTable(64, 64)
    shared = mlora.TokenStep(pool, cache, ws, 4, rope)
    i32 = dict(dtype=torch.int32, device="cuda")
    for T in list(range(1, 34)) + list(range(33, 0, -4)):
        batch = mlora.KVBatch(torch.arange(T, **i32), torch.full((T,), 15, **i32), torch.arange(T, **i32)[:, None])
        x, slots = torch.randn((T, 128), device="cuda", generator=g).half(), torch.randint(-1, 3, (T,), generator=g, **i32)
        alone = mlora.TokenStep(pool, cache, ws, 4, rope)
        for step in (shared, alone):
            step.begin(batch, slots)
        want = alone.layer(0, x).clone()
        got = shared.layer(0, x)
        assert got.shape == (T, 4, 64) and torch.equal(got, want)
    assert len({t.untyped_storage().data_ptr() for k in shared._kept.values() for t in k[2] + [k[3]]}) == 4 * 7


def test_trace_with_prompts():
    """A short trace with keys and values: requests come and go, prompts are shared, every step's attention is that of the cache."""
    H, D, prompt = 256, 64, 40
    times, ids, outs = [0.0, 0.0, 0.05, 0.05, 0.2], [3, 1, 3, 2, 3], [30, 3, 20, 5, 4]
    steps = td.simulate(times, ids, outs, max_prefill_batch_size=2)
    r = td.TraceRunner(2, H, 8, 4, max_batch=8, head_dim=D, prompt=prompt, n_cache_pages=24, dtype=torch.bfloat16)
    seen = 0
    for s in steps:
        if s.kind != "decode" or not len(s.requests):
            continue
        r.decode_step(s.lora_ids, requests=s.requests)
        torch.cuda.synchronize()
        c = r.context
        for layer in range(2):
            q = r.step.qkv[0].view(-1, H // D, D) if layer == 1 else None
            if q is None:
                continue
            for t, (rq, a) in enumerate(zip(s.requests, s.lora_ids)):
                pages = [(p, min(16, prompt - 16 * i)) for i, p in enumerate(c.prompts[int(a)])]
                n = c.length[int(rq)]
                pages += [(p, min(16, n - 16 * i)) for i, p in enumerate(c.pages[int(rq)])]
                for h in (0, 3):
                    kk, vv = (np.concatenate([f64(x[layer, p, h, :m]) for p, m in pages]) for x in (c.cache.k, c.cache.v))
                    want, bound = attention_exact(f64(q[t, h]), kk, vv, D ** -0.5, torch.bfloat16)
                    check(r.attended[layer][t, h], want, bound, f"step {s.index} request {rq}")
                    seen += 1
    assert seen > 40 and max(c.length.values(), default=0) >= 1
    free = c.cache.free_pages
    assert free + sum(map(len, c.pages.values())) + sum(map(len, c.prompts.values())) == 24
