"""What the operators around the LoRA apply refuse before they launch anything: no GPU is needed."""
import ctypes as C

import pytest
import torch

import mlora
from mlora import _ext

one = C.c_void_p(16)          # never dereferenced: every call below fails validation first
off = C.c_void_p(8)
OK, EINVAL, ERANGE, EALIGN, EDTYPE, ENOSPACE = (_ext.MLORA_OK, _ext.MLORA_EINVAL, _ext.MLORA_ERANGE, _ext.MLORA_EALIGN,
                                                _ext.MLORA_EDTYPE, _ext.MLORA_ENOSPACE)


def ptrs(*v):
    return (C.c_void_p * 8)(*(v or (16,) * 8))


def ints(*v):
    return (C.c_int32 * 8)(*(v * 8 if len(v) == 1 else v))


# ---------------------------------------------------------------- 4-bit weights
def gemv(**kw):
    a = dict(n=2, y=ptrs(), x=ptrs(), w=ptrs(), hin=ints(64), hout=ints(64), group=ints(32), zeros=ints(0), T=3, dtype=0)
    a.update(kw)
    return _ext.lib().mlora_w4_gemv_multi(a["n"], a["y"], a["x"], a["w"], a["hin"], a["hout"], a["group"], a["zeros"], a["T"], a["dtype"], 0, None)


@pytest.mark.parametrize("kw, code", [
    (dict(T=0), OK), (dict(dtype=2), EDTYPE), (dict(n=0), ERANGE), (dict(n=9), ERANGE), (dict(T=-1), ERANGE), (dict(T=(1 << 20) + 1), ERANGE),
    (dict(y=None), EINVAL), (dict(group=None), EINVAL), (dict(hin=ints(60)), EALIGN), (dict(hout=ints(63)), EALIGN), (dict(hin=ints(0)), EINVAL),
    (dict(hout=ints(-8)), EINVAL), (dict(group=ints(16)), ERANGE), (dict(group=ints(256)), ERANGE), (dict(y=ptrs(16, 0)), EINVAL),
    (dict(x=ptrs(16, 8)), EALIGN), (dict(w=ptrs(8)), EALIGN), (dict(hin=ints((1 << 24) + 8)), ERANGE),
    (dict(x=ptrs(1 << 20), y=ptrs(1 << 20)), EINVAL), (dict(x=ptrs(1 << 20), y=ptrs((1 << 20) + 16)), EINVAL)])
def test_gemv_arguments(kw, code):
    assert gemv(**kw) == code


def test_pack_arguments():
    lib = _ext.lib()
    need = lib.mlora_w4_packed_bytes(72, 24, 64, 1)
    assert need == 2 * 1 * 1024 + 2 * 2 * 16 * 4               # two column tiles of one K tile; two groups of 16 columns each
    assert lib.mlora_w4_packed_bytes(72, 24, 64, 0) == need - 2 * 2 * 16 * 2
    assert lib.mlora_w4_packed_bytes(72, 24, 48, 0) == ERANGE and lib.mlora_w4_packed_bytes(71, 24, 64, 0) == EALIGN
    pack = lambda c=one, s=one, z=one, p=one, n=need: lib.mlora_w4_pack(c, s, z, 72, 24, 64, p, n, None)     # noqa: E731
    assert pack(n=need - 1) == ENOSPACE and pack(p=off) == EALIGN
    for kw in (dict(c=None), dict(s=None), dict(p=None)):
        assert pack(**kw) == EINVAL


def test_weight_arguments():
    c, s = torch.zeros((64, 16), dtype=torch.uint8), torch.ones((2, 16), dtype=torch.float16)
    for bad in (lambda: mlora.W4Weight(c.int(), s, group=32), lambda: mlora.W4Weight(c, s.float(), group=32), lambda: mlora.W4Weight(c.view(-1), s)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: mlora.W4Weight(c, s, group=16), lambda: mlora.W4Weight(c, s, group=64), lambda: mlora.W4Weight(c, s, s, group=32),
                lambda: mlora.W4Weight(c, s, c, group=32), lambda: mlora.W4Weight(c, s, group=32)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_ext.MloraError):
        mlora.W4Weight(c[:, :12], s[:, :12], group=32)
    with pytest.raises(ValueError):
        mlora.w4_quantize(torch.zeros((8, 8), dtype=torch.float16), group=48)
    with pytest.raises(TypeError):
        mlora.w4_quantize(torch.zeros((8, 8)), group=32)


def test_quantizer_codes_scales_and_a_group_of_zeros():
    w = torch.zeros((40, 8), dtype=torch.float16)
    w[0, 0], w[1, 0], w[35, 1] = 7.0, -7.0, 0.5
    codes, scales, zeros = mlora.w4_quantize(w, 32)
    assert zeros is None and scales.shape == (2, 8) and float(scales[0, 0]) == 1.0 and float(scales[0, 1]) == 0.0
    assert int(codes[0, 0]) == 15 and int(codes[1, 0]) == 1 and (codes[2:, 0] == 8).all() and (codes[:32, 1] == 8).all()
    codes, scales, zeros = mlora.w4_quantize(w, 32, symmetric=False)
    assert int(codes[35, 1]) == 15 and int(zeros[1, 1]) == 0 and int(codes[36, 1]) == 0


# ---------------------------------------------------------------- append
def append(**kw):
    a = dict(q=one, qs=512, o=one, os=512, k=one, ks=128, v=one, vs=128, kp=one, vp=one, n_pages=4, P=16, Hq=8, Hkv=2, D=64, req=one, pos=one, T=3,
             tbl=one, n_req=2, mp=3, of=None, pl=None, n_prefix=0, cs=one, n_pos=9, rot=64, dtype=0)
    a.update(kw)
    return _ext.lib().mlora_kv_append(a["q"], a["qs"], a["o"], a["os"], a["k"], a["ks"], a["v"], a["vs"], a["kp"], a["vp"], a["n_pages"], a["P"], a["Hq"],
                                      a["Hkv"], a["D"], a["req"], a["pos"], a["T"], a["tbl"], a["n_req"], a["mp"], a["of"], a["pl"], a["n_prefix"],
                                      a["cs"], a["n_pos"], a["rot"], 0, None, a["dtype"], None)


@pytest.mark.parametrize("kw, code", [
    (dict(T=0), OK), (dict(dtype=5), EDTYPE), (dict(T=-1), EINVAL), (dict(D=96), ERANGE), (dict(P=8), EINVAL), (dict(P=24), EINVAL), (dict(P=512), EINVAL),
    (dict(n_pages=0), ERANGE), (dict(Hq=7), EINVAL), (dict(Hkv=0), ERANGE), (dict(rot=8), ERANGE), (dict(rot=80), ERANGE), (dict(cs=None), EINVAL),
    (dict(n_pos=0), EINVAL), (dict(k=None), EINVAL), (dict(vp=None), EINVAL), (dict(o=None), EINVAL), (dict(q=None), EINVAL), (dict(k=off), EALIGN),
    (dict(cs=off), EALIGN), (dict(ks=120), EINVAL), (dict(vs=132), EALIGN), (dict(qs=504), EINVAL), (dict(os=520), EINVAL), (dict(req=None), EINVAL),
    (dict(tbl=None), EINVAL), (dict(n_req=0), EINVAL), (dict(mp=0), EINVAL), (dict(mp=1 << 27), ERANGE), (dict(n_prefix=1), EINVAL),
    (dict(n_prefix=-1), ERANGE), (dict(n_prefix=4097), ERANGE), (dict(T=2 ** 31 - 1), ERANGE)])
def test_append_arguments(kw, code):
    assert append(**kw) == code


# ---------------------------------------------------------------- attention
def plan(**kw):
    a = dict(req=one, pos=one, T=3, n_req=2, mp=4, of=None, pl=None, n_prefix=0, mpp=0, P=16, Hq=8, Hkv=2, D=64, buf=one, n=1 << 30)
    a.update(kw)
    return _ext.lib().mlora_attn_plan(a["req"], a["pos"], a["T"], a["n_req"], a["mp"], a["of"], a["pl"], a["n_prefix"], a["mpp"], a["P"], a["Hq"], a["Hkv"], a["D"],
                                      a["buf"], a["n"], None)


@pytest.mark.parametrize("kw, code", [
    (dict(T=0), OK), (dict(T=-1), ERANGE), (dict(T=8193), ERANGE), (dict(n_req=0), EINVAL), (dict(mp=0), EINVAL), (dict(mp=1 << 27), ERANGE),
    (dict(n_prefix=1, mpp=1), EINVAL), (dict(n_prefix=1, of=one, pl=one), EINVAL), (dict(P=20), EINVAL), (dict(Hq=9), EINVAL), (dict(buf=None), EINVAL),
    (dict(buf=off), EALIGN), (dict(n=8), ENOSPACE), (dict(req=None), EINVAL), (dict(D=96), ERANGE)])
def test_plan_arguments(kw, code):
    assert plan(**kw) == code


def attention(**kw):
    a = dict(o=one, os=512, q=one, qs=512, kp=one, vp=one, n_pages=4, P=16, Hq=8, Hkv=2, D=64, req=one, pos=one, T=3, tbl=one, n_req=2, mp=4, of=None,
             pt=None, pl=None, n_prefix=0, mpp=0, plan=one, pn=1 << 30, ws=one, wn=1 << 40, dtype=1, scale=0.1)
    a.update(kw)
    return _ext.lib().mlora_prefix_attention(a["o"], a["os"], a["q"], a["qs"], a["kp"], a["vp"], a["n_pages"], a["P"], a["Hq"], a["Hkv"], a["D"], a["req"],
                                             a["pos"], a["T"], a["tbl"], a["n_req"], a["mp"], a["of"], a["pt"], a["pl"], a["n_prefix"], a["mpp"], a["scale"],
                                             a["plan"], a["pn"], a["ws"], a["wn"], a["dtype"], None)


@pytest.mark.parametrize("kw, code", [
    (dict(T=0), OK), (dict(dtype=3), EDTYPE), (dict(T=-1), ERANGE), (dict(T=9000), ERANGE), (dict(D=80), ERANGE), (dict(Hq=6, Hkv=4), EINVAL),
    (dict(n_pages=-1), ERANGE), (dict(q=None), EINVAL), (dict(o=off), EALIGN), (dict(qs=500), EINVAL), (dict(os=516), EALIGN), (dict(plan=None), EINVAL),
    (dict(pn=8), ENOSPACE), (dict(wn=8), ENOSPACE), (dict(ws=None), ENOSPACE), (dict(n_prefix=2, of=one, pl=one), EINVAL),
    (dict(n_prefix=2, of=one, pl=one, pt=one), EINVAL), (dict(tbl=None), EINVAL), (dict(mp=0), EINVAL), (dict(scale=float("nan")), EINVAL),
    (dict(scale=float("inf")), EINVAL), (dict(scale=float("-inf")), EINVAL)])
def test_attention_arguments(kw, code):
    assert attention(**kw) == code


def test_sizes_grow_with_the_batch():
    """A buffer that was sized for a batch serves every smaller one."""
    lib = _ext.lib()
    for heads, kv in ((1, 1), (32, 32), (32, 8), (64, 1), (40, 8)):
        last = (0, 0)
        for T, n_prefix in ((1, 0), (1, 1), (7, 1), (8, 7), (64, 7), (65, 64), (1000, 64), (8192, 4096)):
            now = (lib.mlora_attn_plan_bytes(T, n_prefix, heads, kv), lib.mlora_attn_workspace_bytes(T, n_prefix, heads, kv, 64))
            assert now[0] >= last[0] and now[1] >= last[1]
            assert lib.mlora_attn_workspace_bytes(T, n_prefix, heads, kv, 128) >= now[1]
            last = now


# ---------------------------------------------------------------- the Python layer
def cache(**kw):
    return mlora.KVCache(**{**dict(n_layers=2, n_pages=4, n_kv_heads=2, head_dim=64, device="cpu"), **kw})


@pytest.mark.parametrize("kw", [dict(head_dim=80), dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=512), dict(n_pages=0), dict(n_kv_heads=0)])
def test_cache_arguments(kw):
    with pytest.raises(ValueError):
        cache(**kw)


def test_cache_pages():
    c = cache(n_pages=5)
    a = c.allocate(3)
    assert len(set(a)) == 3 and c.free_pages == 2
    with pytest.raises(MemoryError):
        c.allocate(3)
    with pytest.raises(ValueError):
        c.release([a[0], a[0]])
    with pytest.raises(ValueError):
        c.release([next(p for p in range(5) if p not in a)])
    c.release(a[:2])
    with pytest.raises(ValueError):
        c.release(a[:1])
    assert c.free_pages == 4 and sorted(c.allocate(4) + a[2:]) == list(range(5))
    with pytest.raises(TypeError):
        cache(dtype=torch.float32)


@pytest.mark.parametrize("kw", [dict(n_pos=0), dict(rot=0), dict(rot=24), dict(rot=256), dict(frequencies=torch.ones(5))])
def test_rope_arguments(kw):
    with pytest.raises(ValueError):
        mlora.RopeTable(**{**dict(n_pos=4, rot=32, device="cpu"), **kw})


def test_rope_table_values():
    t = mlora.RopeTable(100001, 64, device="cpu")
    a = 100000 * torch.tensor(10000.0, dtype=torch.float64) ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    want = torch.cat((torch.cos(a), torch.sin(a))).float()
    assert torch.equal(t.cos_sin[100000], want) and t.cos_sin.shape == (100001, 64)


def test_host_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    batch = mlora.KVBatch(i, i, i.view(1, 2))
    x = torch.zeros((2, 2, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="device tensors"):
        mlora.kv_append(x, x, x, cache(), 0, batch, None)
    with pytest.raises(ValueError, match="device tensors"):
        mlora.plan_attention(batch, cache(), 4)
    with pytest.raises(ValueError, match="device tensors"):
        mlora.prefix_attention(x, cache(), 0, mlora.AttnPlan(batch, 2, 2, 2, 16, torch.zeros(64, dtype=torch.uint8)))
    with pytest.raises(ValueError, match="multiple"):
        mlora.plan_attention(batch, cache(), 3)
    y = torch.zeros((2, 16), dtype=torch.float16)
    with pytest.raises(ValueError, match="device tensors"):
        mlora.w4_gemv([y], [y], [object()])
    with pytest.raises(ValueError, match="1..8"):
        mlora.w4_gemv([], [], [])


# ---------------------------------------------------------------- the step, and the trace's bookkeeping
def test_token_step_arguments():
    pool = mlora.AdapterPool(2, {"q": (64, 256), "k": (64, 128), "v": (64, 128)}, 2, 4, max_rank=16, device="cpu")
    c = cache()
    mlora.TokenStep(pool, c, None, 4)
    with pytest.raises(ValueError, match="q must be"):
        mlora.TokenStep(pool, c, None, 2)
    with pytest.raises(ValueError, match="names"):
        mlora.TokenStep(pool, c, None, 4, names=("q", "k"))
    with pytest.raises(ValueError, match="one dtype"):
        mlora.TokenStep(pool, cache(dtype=torch.bfloat16), None, 4)
    with pytest.raises(ValueError, match="one dtype"):
        mlora.TokenStep(pool, cache(n_layers=1), None, 4)
    with pytest.raises(ValueError, match="every layer"):
        mlora.TokenStep(pool, c, [{}], 4)
    step = mlora.TokenStep(pool, c, None, 4)
    with pytest.raises(RuntimeError, match="begin"):
        step.layer(0, torch.zeros((1, 64), dtype=torch.float16))
    with pytest.raises(ValueError, match="every token"):
        step.begin(mlora.KVBatch(torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros((2, 1), dtype=torch.int32)),
                   torch.zeros(3, dtype=torch.int32))


def test_trace_context_pages():
    from mlora.trace_driver import TraceContext, simulate
    c = TraceContext(mlora.KVCache(1, 12, 1, 64, device="cpu"), 17)
    b = c.advance([5, 9], [2, 2])
    assert b["req_prefix"] == [0, 0] and b["prefix_len"] == [17] and b["tok_pos"] == [17, 17] and len(c.prompts[2]) == 2
    for _ in range(16):
        b = c.advance([5, 9], [2, 2])
    assert b["tok_pos"] == [33, 33] and len(b["pages"][0]) == 2 and c.cache.free_pages == 12 - 2 - 4
    b = c.advance([9, 7], [2, 4])                     # 5 is gone, 7 came with another adapter
    assert b["req_prefix"] == [0, 1] and b["tok_pos"] == [34, 17] and b["pages"][1][1] == -1 and c.cache.free_pages == 12 - 4 - 2 - 1
    for requests, adapters in (([9, 9], [2, 2]), ([9, 7], [2])):
        with pytest.raises(ValueError, match="listed once"):
            c.advance(requests, adapters)
    with pytest.raises(MemoryError):
        c.advance(range(20, 40), [2] * 20)
    steps = simulate([0.0, 0.0, 0.1], [1, 2, 3], [4, 2, 3])
    for s in steps:
        assert len(s.requests) == len(s.lora_ids) and [[1, 2, 3][r] for r in s.requests] == s.lora_ids.tolist()
