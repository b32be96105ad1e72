"""Attention over the paged cache against the 64-bit softmax, with NaN and infinities wherever no key lies."""
import numpy as np
import pytest
import torch

import mlora
from gpu_common import say
from step_ref import U32, Scene, f64, store_bound

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def run(scene, layer=0, scale=None, tokens=None, heads=None, what=""):
    plan = mlora.plan_attention(scene.batch, scene.cache, scene.heads)
    out = torch.full(scene.q.shape, 9.0, dtype=scene.dtype, device="cuda")
    mlora.prefix_attention(scene.dev_q, scene.cache, layer, plan, scale=scale, out=out)
    torch.cuda.synchronize()
    scene.compare(out, layer, scale, tokens, heads, what)
    none = [t for t, r in enumerate(scene.req) if r < 0]
    assert (out[none] == 9.0).all()
    return out, plan


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 127, 128, 129, 500])
def test_one_request(n, D, dtype):
    say(f"attention one request n={n} D={D} {dtype}")
    run(Scene([(-1, n)], [], 4, 2, D, 16, dtype, seed=n))


@pytest.mark.parametrize("heads, kv", [(1, 1), (4, 4), (8, 2), (5, 1), (16, 1), (17, 1), (40, 2), (71, 1)])
def test_head_layouts(heads, kv):
    say(f"attention heads {heads}/{kv}")
    run(Scene([(-1, 70), (0, 5), (0, 40), (0, 1)], [90], heads, kv, 64, 16, F16, seed=heads))


@pytest.mark.parametrize("P", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes(P, D):
    say(f"attention pages of {P} D={D}")
    run(Scene([(0, 37), (0, 300), (-1, 129), (1, 1), (1, 64)], [65, 257], 4, 2, D, P, BF16, seed=P))


@pytest.mark.parametrize("prefix", [1, 15, 16, 31, 33, 100, 128, 1000])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_one_prefix(prefix, dtype):
    """A prefix under several requests, each with keys of its own from one on."""
    say(f"attention prefix={prefix} {dtype}")
    run(Scene([(0, n) for n in (1, 2, 30, 70, 16, 33, 5, 64, 200)], [prefix], 8, 2, 128, 16, dtype, seed=prefix))


@pytest.mark.parametrize("n_req", [2, 3, 16, 17, 40, 65])
def test_group_sizes(n_req):
    """One prefix under as many rows as fill tiles of query rows and one more; requests in no order."""
    say(f"attention group of {n_req}")
    rng = np.random.default_rng(n_req)
    s = Scene([(0, int(rng.integers(1, 40))) for _ in range(n_req)], [300], 8, 4, 64, 16, F16, seed=n_req,
              order=[int(i) for i in rng.permutation(n_req)])
    run(s)


def test_many_prefixes_and_rows_without_a_request():
    say("attention many prefixes")
    rng = np.random.default_rng(5)
    prefixes = [100, 40, 17, 1, 333, 64]
    reqs = [(int(rng.integers(-1, 6)), int(rng.integers(1, 150))) for _ in range(50)]
    run(Scene(reqs, prefixes, 4, 2, 128, 32, BF16, seed=5, pad_rows=(0, 7, 20, 52), order=[int(i) for i in rng.permutation(50)]))


def test_unused_prefixes_and_requests():
    say("attention unused prefixes")
    s = Scene([(2, 10), (2, 20), (-1, 30)], [50, 60, 70, 80], 4, 2, 64, 16, F16, seed=1)
    run(s)


def test_only_rows_without_a_request():
    s = Scene([(-1, 5)], [], 4, 2, 64, 16, F16, seed=1, pad_rows=(1, 2), order=[])
    out, _ = run(s)
    assert (out == 9.0).all()


def test_long_context():
    say("attention long")
    run(Scene([(-1, 20011), (0, 9000), (0, 3)], [5001], 8, 2, 128, 16, BF16, seed=2), heads=[0, 3, 7])


def test_layers_and_scale():
    say("attention layers")
    s = Scene([(0, 20), (0, 50)], [40], 4, 2, 64, 16, F16, seed=3, layers=3)
    for layer in (0, 2):
        run(s, layer=layer)
    run(s, layer=1, scale=0.7)
    run(s, layer=1, scale=-0.3)
    run(s, layer=1, scale=0.0)


def test_peaked_rows():
    """Scores far apart: one key takes the whole weight, in any place of the context."""
    say("attention peaked")
    run(Scene([(0, 100), (-1, 700), (0, 1)], [200], 4, 2, 128, 16, F16, seed=4, std_q=30.0))


@pytest.mark.parametrize("dtype, power", [(F16, 14), (BF16, 40)])
@pytest.mark.parametrize("n_req, D", [(3, 64), (70, 128)])
def test_scores_far_beyond_24_bits(n_req, D, dtype, power):
    """Powers of two, so that every score is exact: the largest key has the whole weight, or shares it with its equals."""
    say(f"attention scores of 2^{2 * power + 6} {dtype}")
    s = Scene([(0, 5 + 7 * i) for i in range(n_req)], [900], 2, 1, D, 16, dtype, seed=n_req)
    g = torch.Generator().manual_seed(5)
    factor = torch.tensor([0.25, 0.5, 1.0])[torch.randint(0, 3, s.k.shape[:4] + (1,), generator=g)].expand(s.k.shape)
    s.k = torch.where(s.k.isnan(), s.k, (factor * 2.0 ** power).to(dtype))
    s.cache.k.copy_(s.k)
    sign = torch.randint(0, 2, (n_req, 2, 1), generator=g) * 2 - 1
    s.q = (sign * 2.0 ** power).expand(n_req, 2, D).to(dtype).contiguous()
    s.dev_q = s.q.cuda()
    plan = mlora.plan_attention(s.batch, s.cache, 2)
    out = f64(mlora.prefix_attention(s.dev_q, s.cache, 0, plan))
    for t in range(n_req):
        k = np.concatenate([s.rows("k", 0, s.prefix_lists[0], 900, 0), s.rows("k", 0, s.req_lists[t], 5 + 7 * t, 0)])
        v = np.concatenate([s.rows("v", 0, s.prefix_lists[0], 900, 0), s.rows("v", 0, s.req_lists[t], 5 + 7 * t, 0)])
        for h in range(2):
            score = k @ f64(s.q[t, h])
            top = v[score == score.max()]
            # n weights of one: fp32 sums of n values in any order, the quotient, the rounding of the result
            bound = (len(top) + 2) * U32 * np.abs(top).sum(0) / len(top) * 1.001 + store_bound(top.mean(0), dtype) * 1.001
            assert (np.abs(out[t, h] - top.mean(0)) <= bound).all(), (t, h)


@pytest.mark.parametrize("n_req", [1, 6, 70])
@pytest.mark.parametrize("prefix, own", [(0, 20), (0, 3000), (400, 30)])
def test_a_nan_query_stays_nan_and_alone(n_req, prefix, own):
    """One head of one token is NaN: it has no maximum, cut into parts or not.  The rows beside it in its tile are what they are without it."""
    say(f"attention NaN query, {n_req} requests, prefix {prefix}, own {own}")
    s = Scene([(0 if prefix else -1, own + i % 5) for i in range(n_req)], [prefix] if prefix else [], 4, 2, 64, 16, BF16, seed=own)
    plan = mlora.plan_attention(s.batch, s.cache, 4)
    want = mlora.prefix_attention(s.dev_q, s.cache, 0, plan)
    t = n_req // 2
    s.dev_q[t, 1] = float("nan")
    got = mlora.prefix_attention(s.dev_q, s.cache, 0, plan)
    assert got[t, 1].isnan().all()
    got[t, 1] = want[t, 1]
    assert torch.equal(got, want)


def test_positions_inside_the_prefix_and_before_the_start():
    """A token at a position of its own prefix sees the prefix up to itself; one before the start sees nothing and is zeros."""
    say("attention positions inside the prefix")
    s = Scene([(0, 10), (0, 20), (0, 30), (-1, 40), (-1, 50)], [100], 4, 2, 64, 16, F16, seed=6)
    s.pos = [37, 99, 129, -1, 0]
    s.batch.tok_pos.copy_(torch.tensor(s.pos, dtype=torch.int32))
    out, _ = run(s)
    assert (out[3] == 0).all()


def test_several_tokens_of_one_request():
    say("attention several tokens of a request")
    s = Scene([(0, 40), (-1, 50)], [70], 8, 2, 128, 16, BF16, seed=7)
    s.req, s.pos = [0, 0, 1, 0, 1], [70, 109, 49, 100, 3]
    s.batch.tok_req = torch.tensor(s.req, dtype=torch.int32, device="cuda")
    s.batch.tok_pos = torch.tensor(s.pos, dtype=torch.int32, device="cuda")
    s.q = torch.randn((5, 8, 128)).to(BF16)
    s.dev_q = s.q.cuda()
    run(s)


@pytest.mark.parametrize("bad", [-1, 10 ** 6, -(2 ** 31), 2 ** 31 - 1])
def test_keys_on_bad_pages_are_absent(bad):
    say(f"attention bad page {bad}")
    s = Scene([(0, 100), (0, 60), (-1, 200), (-1, 10)], [90], 4, 2, 64, 16, F16, seed=8)
    for lists, table in ((s.req_lists, s.batch.pages), (s.prefix_lists, s.batch.prefix_pages)):
        for row, col in (((0, 2), (2, 0), (3, 0)) if lists is s.req_lists else ((0, 3),)):
            lists[row][col] = bad
            table[row, col] = bad
    out, _ = run(s)
    assert (out[3] == 0).all()


def test_requests_out_of_range_and_positions_behind_the_tables():
    """A request that no table holds sees no key; a position behind the table's end sees the keys that are there."""
    say("attention requests out of range")
    s = Scene([(0, 100), (-1, 64)], [48], 4, 2, 64, 16, F16, seed=9)
    plan_pos = [48 + 99, 2 ** 31 - 1, 5]
    s.batch.tok_req = torch.tensor([0, 1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    s.batch.tok_pos = torch.tensor(plan_pos, dtype=torch.int32, device="cuda")
    # request 1's table is as wide as request 0's: behind its own 64 keys it lists no page
    s.q = torch.randn((3, 4, 64)).to(F16)
    s.dev_q = s.q.cuda()
    plan = mlora.plan_attention(s.batch, s.cache, 4)
    out = torch.full((3, 4, 64), 9.0, dtype=F16, device="cuda")
    mlora.prefix_attention(s.dev_q, s.cache, 0, plan, out=out)
    s.req, s.pos = [0, 1, -1], [147, 63, 0]
    s.compare(out)
    assert (out[2] == 0).all()


def test_views_of_a_wider_output():
    """q and out as rows of wider tensors; what lies between the rows stays."""
    say("attention strided")
    s = Scene([(0, 33), (0, 9), (-1, 80)], [40], 4, 2, 64, 16, F16, seed=10)
    wide = torch.full((3, 10, 64), 7.0, dtype=F16, device="cuda")
    wide[:, 2:6] = s.dev_q
    out = torch.full((3, 9, 64), 5.0, dtype=F16, device="cuda")
    plan = mlora.plan_attention(s.batch, s.cache, 4)
    mlora.prefix_attention(wide[:, 2:6], s.cache, 0, plan, out=out[:, 1:5])
    s.compare(out[:, 1:5])
    assert (out[:, 0] == 5.0).all() and (out[:, 5:] == 5.0).all()


def test_new_output_is_zeros_where_no_request_is():
    s = Scene([(-1, 20)], [], 4, 2, 64, 16, F16, seed=11, pad_rows=(1,))
    plan = mlora.plan_attention(s.batch, s.cache, 4)
    out = mlora.prefix_attention(s.dev_q, s.cache, 0, plan)
    s.compare(out)
    assert (out[1] == 0).all()


def test_a_plan_is_reused_for_smaller_batches():
    say("attention plan reuse")
    big = Scene([(i % 3 - 1, 20 + 7 * i) for i in range(40)], [100, 50], 4, 2, 64, 16, F16, seed=12)
    out, plan = run(big)
    small = Scene([(1, 9), (0, 70), (1, 3)], [33, 200], 4, 2, 64, 16, F16, seed=13)
    plan = mlora.plan_attention(small.batch, small.cache, 4, out=plan)
    got = mlora.prefix_attention(small.dev_q, small.cache, 0, plan)
    small.compare(got)


def test_repeated_calls_give_the_same_bits():
    s = Scene([(0, 33 * (i + 1)) for i in range(20)], [777], 8, 2, 128, 16, BF16, seed=14)
    first, plan = run(s, tokens=[0, 19], heads=[0])
    for _ in range(3):
        assert torch.equal(mlora.prefix_attention(s.dev_q, s.cache, 0, plan), first)


def test_captured_step_replays():
    """Plan and layers captured once; lengths, queries and keys change between replays."""
    say("attention captured")
    s = Scene([(0, 200), (0, 150), (-1, 90), (0, 40)], [130], 8, 2, 64, 16, F16, seed=15)
    plan = mlora.plan_attention(s.batch, s.cache, 8)
    out = torch.zeros_like(s.dev_q)
    mlora.prefix_attention(s.dev_q, s.cache, 0, plan, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mlora.plan_attention(s.batch, s.cache, 8, out=plan)
        mlora.prefix_attention(s.dev_q, s.cache, 0, plan, out=out)
    for i, pos in enumerate([[150, 200, 3, 140], [329, 131, 89, 169], [130, 130, 0, 130], [10, 279, 50, 150]]):
        s.pos = pos
        s.batch.tok_pos.copy_(torch.tensor(pos, dtype=torch.int32))
        s.q = torch.randn(s.q.shape).to(F16)
        s.dev_q.copy_(s.q)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        s.compare(got, what=f"replay {i}")
        mlora.plan_attention(s.batch, s.cache, 8, out=plan)
        mlora.prefix_attention(s.dev_q, s.cache, 0, plan, out=out)
        assert torch.equal(got, out)


def test_calls_that_share_a_plan_on_two_streams():
    s = Scene([(0, 33 * (i + 1)) for i in range(12)], [500], 8, 2, 128, 16, F16, seed=16, layers=2)
    plan = mlora.plan_attention(s.batch, s.cache, 8)
    want = [mlora.prefix_attention(s.dev_q, s.cache, l, plan) for l in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [torch.zeros_like(s.dev_q) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for l, st in enumerate(streams):
            with torch.cuda.stream(st):
                mlora.prefix_attention(s.dev_q, s.cache, l, plan, out=outs[l])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_offsets_past_32_bits():
    """A layer's slab of more than 2^32 elements, keys on its first and last pages."""
    say("attention large slab")
    n_pages = (1 << 32) // (8 * 256 * 128) + 3
    cache = mlora.KVCache(1, n_pages, 8, 128, page_tokens=256, dtype=BF16)
    small = Scene([(-1, 300)], [], 8, 8, 128, 256, BF16, seed=17)
    a, b = small.req_lists[0]
    for new, old in ((n_pages - 1, a), (0, b)):
        cache.k[0, new].copy_(small.cache.k[0, old])
        cache.v[0, new].copy_(small.cache.v[0, old])
    small.batch.pages.copy_(torch.tensor([[n_pages - 1, 0]], dtype=torch.int32))
    plan = mlora.plan_attention(small.batch, cache, 8)
    small.compare(mlora.prefix_attention(small.dev_q, cache, 0, plan))


def test_no_tokens():
    cache = mlora.KVCache(1, 4, 2, 64)
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    batch = mlora.KVBatch(e, e, torch.zeros((1, 1), dtype=torch.int32, device="cuda"))
    plan = mlora.plan_attention(batch, cache, 4)
    assert mlora.prefix_attention(torch.empty((0, 4, 64), dtype=F16, device="cuda"), cache, 0, plan).shape == (0, 4, 64)


def test_refusals():
    s = Scene([(0, 20), (-1, 30)], [40], 4, 2, 64, 16, F16, seed=18, layers=2)
    plan = mlora.plan_attention(s.batch, s.cache, 4)
    q = s.dev_q
    with pytest.raises(IndexError):
        mlora.prefix_attention(q, s.cache, 2, plan)
    with pytest.raises(ValueError, match="q must be"):
        mlora.prefix_attention(q[:1], s.cache, 0, plan)
    with pytest.raises(TypeError, match="dtype"):
        mlora.prefix_attention(q.float(), s.cache, 0, plan)
    with pytest.raises(ValueError, match="behind the other"):
        mlora.prefix_attention(torch.zeros((2, 64, 4), dtype=F16, device="cuda").transpose(1, 2), s.cache, 0, plan)
    with pytest.raises(mlora.MloraError, match="stride"):
        mlora.prefix_attention(q[:1].expand(2, 4, 64), s.cache, 0, plan)
    with pytest.raises(ValueError, match="another cache layout"):
        mlora.prefix_attention(q, mlora.KVCache(1, 4, 4, 64), 0, plan)
    with pytest.raises(ValueError, match="another cache layout"):
        mlora.prefix_attention(q, mlora.KVCache(1, 4, 2, 64, page_tokens=32), 0, plan)
    pages, of = s.batch.pages, s.batch.req_prefix
    s.batch.pages, s.batch.req_prefix = pages[:1].contiguous(), of[:1].contiguous()       # a table that the plan has not seen
    with pytest.raises(ValueError, match="number of requests"):
        mlora.prefix_attention(q, s.cache, 0, plan)
    s.batch.pages, s.batch.req_prefix = pages, of
    many = Scene([(0, 5)] * 400, [40], 4, 2, 64, 16, F16, seed=18)
    with pytest.raises(mlora.MloraError) as e:
        mlora.plan_attention(many.batch, many.cache, 4, out=plan)
    assert e.value.code == mlora._ext.MLORA_ENOSPACE
    s.compare(mlora.prefix_attention(q, s.cache, 0, plan))          # the plan is still the one it was
    for field, value, error in (("tok_pos", s.batch.tok_pos.long(), TypeError), ("tok_pos", s.batch.tok_pos[:1], ValueError),
                                ("pages", s.batch.pages[0], ValueError), ("pages", s.batch.pages.t(), ValueError),
                                ("req_prefix", s.batch.req_prefix[:1], ValueError), ("prefix_len", None, ValueError),
                                ("prefix_pages", None, ValueError), ("prefix_pages", s.batch.prefix_pages.repeat(2, 1), ValueError),
                                ("tok_req", s.batch.tok_req.cpu(), ValueError)):
        old = getattr(s.batch, field)
        setattr(s.batch, field, value)
        with pytest.raises(error):
            mlora.plan_attention(s.batch, s.cache, 4)
        setattr(s.batch, field, old)


@pytest.mark.parametrize("dtype, D, P", [(F16, 128, 16), (BF16, 64, 16), (BF16, 128, 64), (F16, 64, 256)])
@pytest.mark.parametrize("n_req, prefix", [(17, 63), (17, 64), (33, 65), (40, 129), (64, 1000), (65, 1)])
def test_groups_of_many_rows(n_req, prefix, dtype, D, P):
    """From 65 rows on the wavefronts of a workgroup share the rows: full and odd tiles of rows and of keys, absent pages among them."""
    say(f"attention rows {4 * n_req} prefix {prefix} {dtype} D={D} P={P}")
    rng = np.random.default_rng(n_req + prefix)
    s = Scene([(0, int(rng.integers(1, 20))) for _ in range(n_req)], [prefix], 4, 1, D, P, dtype, seed=n_req + prefix)
    if prefix > 2 * P:
        s.prefix_lists[0][1] = -1
        s.batch.prefix_pages[0, 1] = -1
    run(s)
