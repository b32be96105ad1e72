"""What the microscaled products and the page tables refuse before they launch anything: no GPU is needed."""
import ctypes as C

import numpy as np
import pytest
import torch

import mlora
import mx4_ref as ref
from mlora import _ext
from pages_ref import Tables

one = C.c_void_p(16)          # never dereferenced: every call below fails validation first
off = C.c_void_p(8)
OK, EINVAL, ERANGE, EALIGN, EDTYPE, ENOSPACE = (_ext.MLORA_OK, _ext.MLORA_EINVAL, _ext.MLORA_ERANGE, _ext.MLORA_EALIGN,
                                                _ext.MLORA_EDTYPE, _ext.MLORA_ENOSPACE)


def ptrs(*v):
    return (C.c_void_p * 8)(*(v or (16,) * 8))


def ints(*v):
    return (C.c_int32 * 8)(*(v * 8 if len(v) == 1 else v))


# ---------------------------------------------------------------- operands
def test_sizes_of_an_operand():
    size = _ext.lib().mlora_mx4_bytes
    assert size(1, 8) == 1024 + 256 and size(16, 128) == 1024 + 256 and size(17, 520) == 2 * (5 * 1024 + 2 * 256)
    assert size(0, 64) == 0
    assert size(-1, 64) == EINVAL and size(1, 0) == EINVAL and size(1, 12) == EALIGN
    assert size((1 << 24) + 1, 8) == ERANGE and size(1, (1 << 24) + 8) == ERANGE
    assert size(1 << 24, 1 << 24) > 1 << 47


@pytest.mark.parametrize("kw, code", [
    (dict(rows=0), OK), (dict(dtype=2), EDTYPE), (dict(rows=-1), EINVAL), (dict(k=60), EALIGN), (dict(x=None), EINVAL), (dict(x=off), EALIGN),
    (dict(stride=68), EALIGN), (dict(stride=56), EINVAL), (dict(packed=None), EINVAL), (dict(packed=off), EALIGN), (dict(n=1279), ENOSPACE)])
def test_quantize_and_values_arguments(kw, code):
    a = dict(x=one, stride=64, rows=3, k=64, dtype=0, packed=one, n=1280)
    a.update(kw)
    assert _ext.lib().mlora_mx4_quantize(a["x"], a["stride"], a["rows"], a["k"], a["dtype"], a["packed"], a["n"], None) == code
    assert _ext.lib().mlora_mx4_values(a["packed"], a["n"], a["rows"], a["k"], a["x"], a["stride"], a["dtype"], None) == code


@pytest.mark.parametrize("kw, code", [(dict(rows=0), OK), (dict(k=4), EALIGN), (dict(c=None), EINVAL), (dict(s=None), EINVAL), (dict(p=None), EINVAL), (dict(p=off), EALIGN), (dict(n=1279), ENOSPACE)])
def test_pack_arguments(kw, code):
    a = dict(c=one, s=one, rows=3, k=64, p=one, n=1280)
    a.update(kw)
    assert _ext.lib().mlora_mx4_pack(a["c"], a["s"], a["rows"], a["k"], a["p"], a["n"], None) == code


# 3 rows of 64 columns, 80 elements apart: 448 bytes; packed 1280, codes 96, scales 6
@pytest.mark.parametrize("at", [1 << 20, (1 << 20) + 432, (1 << 20) - 1264])
def test_operands_that_overlap_their_source(at):
    lib, rows, packed = _ext.lib(), C.c_void_p(1 << 20), C.c_void_p(at)
    assert lib.mlora_mx4_quantize(rows, 80, 3, 64, 0, packed, 1280, None) == EINVAL
    assert lib.mlora_mx4_values(packed, 1280, 3, 64, rows, 80, 1, None) == EINVAL
    near = C.c_void_p(at if at != (1 << 20) + 432 else (1 << 20) + 80)
    assert lib.mlora_mx4_pack(rows, one, 3, 64, near, 1280, None) == EINVAL
    near = C.c_void_p(at if at != (1 << 20) + 432 else 1 << 20)
    assert lib.mlora_mx4_pack(one, rows, 3, 64, near, 1280, None) == EINVAL


def gemm(**kw):
    a = dict(n=2, y=ptrs(1 << 20, 2 << 20, *[16] * 6), x=ptrs(3 << 20, 3 << 20, *[16] * 6), w=ptrs(4 << 20, 5 << 20, *[16] * 6), hin=ints(64), hout=ints(64), T=3, dtype=0)
    a.update(kw)
    return _ext.lib().mlora_mx4_gemm_multi(a["n"], a["y"], a["x"], a["w"], a["hin"], a["hout"], a["T"], a["dtype"], 0, None)


@pytest.mark.parametrize("kw, code", [
    (dict(T=0), OK), (dict(dtype=2), EDTYPE), (dict(n=0), ERANGE), (dict(n=9), ERANGE), (dict(T=-1), ERANGE), (dict(T=(1 << 20) + 1), ERANGE),
    (dict(y=None), EINVAL), (dict(x=None), EINVAL), (dict(w=None), EINVAL), (dict(hin=None), EINVAL), (dict(hout=None), EINVAL), (dict(hin=ints(60)), EALIGN),
    (dict(hout=ints(63)), EALIGN), (dict(hin=ints(0)), EINVAL), (dict(hout=ints(0)), EINVAL), (dict(hout=ints(-8)), EINVAL), (dict(hin=ints((1 << 24) + 8)), ERANGE),
    (dict(hout=ints((1 << 24) + 8)), ERANGE), (dict(y=ptrs(1 << 20, 0)), EINVAL), (dict(x=ptrs(3 << 20, 8)), EALIGN), (dict(w=ptrs(8)), EALIGN),
    (dict(y=ptrs(1 << 20, 1 << 20)), EINVAL), (dict(y=ptrs(1 << 20, (3 << 20) + 1264)), EINVAL), (dict(y=ptrs((4 << 20) + 16, 2 << 20)), EINVAL)])
def test_gemm_arguments(kw, code):
    assert gemm(**kw) == code


def test_form_arguments():
    form, shape = _ext.lib().mlora_mx4_form, (C.c_int32 * 2)()
    assert form(1, ints(4096), ints(4096), 1, shape) == OK and list(shape) == [16, 16]
    assert form(2, ints(5120), ints(13824), 8000, shape) == OK and list(shape) == [256, 256]
    assert form(1, ints(64), ints(64), 1 << 20, shape) == OK and form(8, ints(1 << 24), ints(1 << 24), 1 << 20, shape) == OK
    assert form(0, ints(64), ints(64), 1, shape) == ERANGE and form(1, ints(60), ints(64), 1, shape) == EALIGN
    assert form(1, ints(64), ints(64), 0, shape) == EINVAL and form(1, ints(64), ints(64), 1, None) == EINVAL


def test_operands_from_python():
    c, s = torch.zeros((16, 32), dtype=torch.uint8), torch.zeros((16, 2), dtype=torch.uint8)
    for bad in (lambda: mlora.MX4Tensor(c.int(), s), lambda: mlora.MX4Tensor(c, s.int()), lambda: mlora.MX4Tensor(c.view(-1), s)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: mlora.MX4Tensor(c, s[:, :1]), lambda: mlora.MX4Weight(c, s[:8]), lambda: mlora.MX4Tensor(c, s), lambda: mlora.mx4_quantize(torch.zeros(8).half()),
                lambda: mlora.mx4_quantize(torch.zeros((2, 8)).half()), lambda: mlora.MX4Weight.quantize(torch.zeros(8).half())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        mlora.mx4_quantize(torch.zeros((2, 8)))
    with pytest.raises(_ext.MloraError):
        mlora.MX4Tensor(c[:, :31], s)
    with pytest.raises(ValueError):
        mlora.mx4_gemm([], [], [])


# ---------------------------------------------------------------- page tables
def layout(n_req=4, max_pages=5, n_pages=70):
    at = (C.c_int64 * _ext.PAGES_LAYOUT_WORDS)()
    return _ext.lib().mlora_pages_layout(n_req, max_pages, n_pages, at), list(at)


def test_layout():
    rc, at = layout()
    assert rc == OK and at[:7] == [0, 32, 52, 56, 126, 127, 128] and at[7] >= 32 + 2 + 4 * 70
    for kw, code in ((dict(n_req=0), EINVAL), (dict(max_pages=0), EINVAL), (dict(n_pages=0), EINVAL), (dict(n_pages=(1 << 24) + 1), ERANGE),
                     (dict(n_req=1 << 16, max_pages=(1 << 14) + 1), ERANGE), (dict(n_req=(1 << 20) + 1), ERANGE)):
        assert layout(**kw)[0] == code
    assert _ext.lib().mlora_pages_layout(1, 1, 1, None) == EINVAL


@pytest.mark.parametrize("kw, code", [
    (dict(state=None), EINVAL), (dict(scratch=None), EINVAL), (dict(want=None), EINVAL), (dict(state=off), EALIGN), (dict(scratch=off), EALIGN),
    (dict(words=127), ENOSPACE), (dict(scratch_words=200), ENOSPACE), (dict(n_req=0), EINVAL), (dict(max_pages=-1), EINVAL), (dict(n_pages=0), EINVAL),
    (dict(P=8), EINVAL), (dict(P=48), EINVAL), (dict(P=512), EINVAL), (dict(max_pages=1 << 27, n_req=1), ERANGE),
    (dict(k=None), EINVAL), (dict(v=None), EINVAL), (dict(k=off), EALIGN), (dict(layers=0), EINVAL), (dict(heads=0), EINVAL), (dict(D=96), ERANGE),
    (dict(heads=(1 << 14) + 1), ERANGE)])
def test_page_calls(kw, code):
    lib = _ext.lib()
    a = dict(state=one, words=1 << 20, scratch=one, scratch_words=1 << 20, want=C.c_void_p(1 << 30), n_req=4, max_pages=5, n_pages=70, P=16, k=one, v=one, layers=2, heads=2, D=64)
    a.update(kw)
    slabs = (a["k"], a["v"], a["layers"], a["n_pages"], a["heads"], a["P"], a["D"])
    assert lib.mlora_pages_resize(a["state"], a["words"], a["scratch"], a["scratch_words"], a["want"], a["n_req"], a["max_pages"], *slabs, None) == code
    if "want" not in kw:
        assert lib.mlora_pages_compact(a["state"], a["words"], a["scratch"], a["scratch_words"], a["n_req"], a["max_pages"], *slabs, None) == code
    if not {"k", "v", "layers", "heads", "D"} & set(kw):
        assert lib.mlora_pages_fork(a["state"], a["words"], a["scratch"], a["scratch_words"], a["want"], a["n_req"], a["max_pages"], a["n_pages"], a["P"], None) == code


def test_rows_values_inside_the_tables():
    """Lengths given as the tables' own would never differ from them, and parents there would change under the call."""
    lib, state, scratch = _ext.lib(), 1 << 20, 1 << 24
    for want in (state, state + 56 * 4, state - 12, scratch + 4 * 127):
        assert lib.mlora_pages_resize(C.c_void_p(state), 128, C.c_void_p(scratch), 1 << 16, C.c_void_p(want), 4, 5, one, one, 2, 70, 2, 16, 64, None) == EINVAL
        assert lib.mlora_pages_fork(C.c_void_p(state), 128, C.c_void_p(scratch), 1 << 16, C.c_void_p(want), 4, 5, 70, 16, None) == EINVAL
        assert b"must not lie" in lib.mlora_last_error()


def host_pages(n_req=3, max_pages=4, n_pages=20, taken=None):
    cache = mlora.KVCache(1, n_pages, 1, 64, device="cpu")
    return cache, mlora.KVPages(cache, n_req, max_pages, taken)


def test_pages_from_python():
    cache, p = host_pages()
    assert cache.free_pages == 0 and p.table.tolist() == [[-1] * 4] * 3 and p.lens.tolist() == [0] * 3 and p.refs.tolist() == [0] * 20
    for call in (p.resize, p.fork):
        with pytest.raises(ValueError):
            call(torch.zeros(3, dtype=torch.int32))            # not on the device
    with pytest.raises(ValueError):
        p.compact()
    with pytest.raises(ValueError):
        p.adopt(torch.zeros((3, 5), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(MemoryError):
        mlora.KVPages(cache, 2, 2, 1)
    with pytest.raises(_ext.MloraError):
        mlora.KVPages(cache, 0, 2)
    with pytest.raises(ValueError):
        mlora.KVPages(mlora.KVCache(1, 4, 1, 64, device="cpu"), 1, (1 << 26) + 1)


def test_pages_change_hands_with_the_cache():
    cache, p = host_pages(taken=7)
    assert cache.free_pages == 13
    p.take(3)
    table = torch.tensor([[0, 4, -1, -1], [0, 3, 9, 9], [8, 8, 8, 8]], dtype=torch.int32)
    for lens in ([32, 48, 64], [33, 0, 0], [0, 49, 0], [-1, 0, 0], [0, 0, 65]):
        with pytest.raises(ValueError):
            p.adopt(table, torch.tensor(lens, dtype=torch.int32))
    p.adopt(table, torch.tensor([32, 17, 0], dtype=torch.int32))
    assert p.refs.tolist()[:10] == [2, 0, 0, 1, 1, 0, 0, 0, 0, 0] and p.table.tolist() == [[0, 4, -1, -1], [0, 3, -1, -1], [-1] * 4]
    assert p.give_back() == 5 and cache.free_pages == 15
    with pytest.raises(ValueError):
        p.adopt(torch.full((3, 4), 9, dtype=torch.int32), torch.tensor([1, 0, 0], dtype=torch.int32))
    p.adopt(table, torch.zeros(3, dtype=torch.int32))
    assert p.give_back() == 5 and cache.free_pages == 20


# ---------------------------------------------------------------- the plain forms themselves
def test_grid_ties_and_saturation():
    x = np.zeros((1, 32))
    x[0, :12] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.7499, 0.2501, -7.9]
    codes, scales = ref.quantize(x)
    assert scales.tolist() == [[127]]
    assert ref.values(codes, scales)[0, :12].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -0.0, -0.5, 0.5, -6.0]
    assert ref.quantize(np.full((1, 8), 2.0 ** -133))[1].tolist() == [[0]] and ref.quantize(np.zeros((1, 8)))[1].tolist() == [[0]]
    assert np.isnan(ref.values(*ref.quantize(np.array([[1.0, np.inf]] * 1)))).all()


def test_model_of_the_tables():
    t = Tables([[], []], [0, 0], range(4), 4, 16, 3)
    assert t.resize([17, 16]) == [] and t.rows == [[0, 1], [2]]
    t.fork([-1, 0])
    assert t.rows == [[0, 1], [0, 1]] and t.refs() == [2, 2, 0, 0]
    assert t.resize([18, 18]) == [(1, 2, 1)] and t.rows == [[0, 2], [0, 1]]
    assert t.resize([0, -1]) == [] and t.compact() == [] and t.rows[1] == [0, 1]
