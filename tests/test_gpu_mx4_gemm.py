"""Products of microscaled 4-bit operands against the 64-bit product of the values they stand for."""
import ctypes as C

import numpy as np
import pytest
import torch

import mlora
import mx4_ref as ref
from gpu_common import say
from mlora import _ext
from step_ref import check, store_bound

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def operand(rows, k, seed, spread=3, make=None):
    """A packed operand of random codes whose blocks' powers of two lie within 2^spread of each other, and its values."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (rows, k))
    scales = rng.integers(125 - spread, 126, (rows, -(-k // 32))).astype(np.uint8)
    made = (make or mlora.MX4Tensor)(torch.from_numpy(ref.packed_codes(codes)).cuda(), torch.from_numpy(scales).cuda())
    return made, ref.values(codes, scales)


def compare(y, xv, wv, dtype, y0=None, what=""):
    want, bound = ref.gemm(xv, wv, y0)
    check(y, want, bound + store_bound(np.abs(want) + bound, dtype), what)


def run(T, k, n, dtype, seed=0, accumulate=False, spread=3):
    what = f"mx4_gemm T={T} {k}->{n} {dtype} acc={accumulate}"
    say(what)
    x, xv = operand(T, k, seed, spread)
    w, wv = operand(n, k, seed + 1, spread, mlora.MX4Weight)
    y = torch.randn((T, n), device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)
    y0 = ref.f64(y) if accumulate else None
    mlora.mx4_gemm([y], [x], [w], accumulate=accumulate)
    compare(y, xv, wv, dtype, y0, what)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T, k, n", [(1, 32, 8), (1, 4096, 256), (3, 8, 24), (16, 128, 16), (17, 136, 40), (61, 2048, 200), (130, 520, 264), (300, 1000, 136)])
def test_product(T, k, n, dtype):
    run(T, k, n, dtype)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 48, 49, 63, 64, 65, 96, 97, 127, 128, 129, 192, 193, 255, 256, 257, 400])
def test_numbers_of_tokens(T):
    run(T, 384, 144, BF16, seed=T)


@pytest.mark.parametrize("k", [8, 24, 32, 40, 120, 128, 136, 256, 384, 504, 512, 520, 1024, 2752, 5504, 11008])
def test_input_widths(k):
    """The last block, the last tile and the last quad of tiles end anywhere."""
    run(3, k, 64, F16, seed=k)
    run(70, k, 64, BF16, seed=k)


@pytest.mark.parametrize("n", [8, 16, 24, 56, 64, 72, 120, 128, 136, 248, 256, 264, 1032, 4096])
def test_output_widths(n):
    run(2, 256, n, F16, seed=n)
    run(40, 256, n, F16, seed=n)
    run(260, 256, n, BF16, seed=n)


# the last three: tiles of 256 tokens alone, halves alone, both
FORMS = [((16, 16), 17, 136, 72), ((32, 16), 17, 136, 2056), ((16, 32), 50, 2184, 1032), ((32, 32), 50, 1032, 2056), ((32, 64), 257, 1032, 1032), ((64, 64), 201, 2184, 2056),
         ((128, 64), 300, 136, 2056), ((128, 128), 1030, 136, 2056), ((256, 256), 1030, 2184, 8200), ((256, 256), 1030, 2184, 4104), ((256, 256), 2570, 1160, 8200)]


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("form, T, k, n", FORMS)
def test_every_form(form, T, k, n, dtype, accumulate):
    """Sizes that end inside a block, a tile, a quad of tiles and a workgroup's columns and tokens."""
    shape = (C.c_int32 * 2)()
    assert _ext.lib().mlora_mx4_form(1, (C.c_int32 * 1)(k), (C.c_int32 * 1)(n), T, shape) == 0 and tuple(shape) == form
    run(T, k, n, dtype, accumulate=accumulate)


@pytest.mark.parametrize("k", [8, 128, 256, 384, 512, 640, 768, 896, 1024, 1152, 2176])
def test_steps_of_the_large_tiles(k):
    """Every number of steps on either side of a ring's four stages."""
    say(f"large tiles k={k}")
    for T, n in ((2570, 8200), (1030, 4104), (1030, 2056), (300, 2056)):
        run(T, k, n, BF16, seed=k)


@pytest.mark.parametrize("T", [1, 20, 100, 300])
def test_accumulate(T):
    run(T, 640, 200, F16, accumulate=True)
    run(T, 640, 200, BF16, accumulate=True)


def test_the_most_tokens():
    """2^20 tokens of one narrow product: more rows of workgroups than a launch's second dimension takes, compared at both ends and in the middle."""
    say("mx4_gemm 2^20 tokens")
    T = 1 << 20
    base, xv = operand(64, 40, 1)
    row = base.values(BF16)
    x = mlora.mx4_quantize(row.repeat(T // 64, 1))
    w, wv = operand(8, 40, 2, 3, mlora.MX4Weight)
    y = torch.empty((T, 8), dtype=BF16, device="cuda")
    mlora.mx4_gemm([y], [x], [w])
    again = ref.values(*ref.quantize(xv))
    for at in (0, T // 2, T - 64):
        compare(y[at:at + 64], again, wv, BF16, what=f"rows from {at}")
    assert torch.equal(y.view(-1, 64, 8), y[:64].expand(T // 64, 64, 8))


def test_powers_of_two_far_apart():
    """Blocks whose scales differ by up to 2^40: the small ones fall below what fp32 holds beside the large ones."""
    run(20, 1024, 64, BF16, spread=40)
    run(300, 1024, 264, BF16, spread=40)


@pytest.mark.parametrize("T", [1, 33, 200, 513])
def test_projections_of_one_call(T):
    """Different widths and inputs in one call, some of them shared."""
    say(f"mx4_gemm projections T={T}")
    xa, va = operand(T, 512, 1)
    xb, vb = operand(T, 392, 2)
    sizes = [(512, 256, xa, va), (512, 72, xa, va), (392, 1032, xb, vb), (512, 8, xa, va), (392, 144, xb, vb)]
    ws = [operand(n, k, 10 + i, 3, mlora.MX4Weight) for i, (k, n, _, _) in enumerate(sizes)]
    ys = [torch.empty((T, n), dtype=F16, device="cuda") for _, n, _, _ in sizes]
    mlora.mx4_gemm(ys, [s[2] for s in sizes], [w for w, _ in ws])
    for y, s, (_, wv) in zip(ys, sizes, ws):
        compare(y, s[3], wv, F16, what=f"{s[0]}->{s[1]}")


def test_nan_stays_in_its_row_and_column():
    say("mx4_gemm NaN")
    for T in (5, 40, 300):
        k, n = 640, 264
        x = torch.randn((T, k), generator=torch.Generator().manual_seed(T)).to(BF16)
        x[3, 100] = float("inf")
        q = mlora.mx4_quantize(x.cuda())
        codes, scales = np.random.default_rng(T).integers(0, 16, (n, k)), np.full((n, 20), 120, np.uint8)
        codes[8, 32:64], scales[8, 1] = 0, 255
        w = mlora.MX4Weight(torch.from_numpy(ref.packed_codes(codes)).cuda(), torch.from_numpy(scales).cuda())
        y = torch.empty((T, n), dtype=BF16, device="cuda")
        mlora.mx4_gemm([y], [q], [w])
        nan = torch.zeros((T, n), dtype=torch.bool)
        nan[3], nan[:, 8] = True, True
        assert torch.equal(torch.isnan(y).cpu(), nan)


def test_quantised_input_and_weight_end_to_end():
    """As a layer calls it: 16-bit rows and weight in, quantised, multiplied."""
    say("mx4 linear")
    g = torch.Generator().manual_seed(9)
    x, w = torch.randn((77, 1024), generator=g).to(F16), (torch.randn((1024, 328), generator=g) * 0.02).to(F16)
    y = torch.empty((77, 328), dtype=F16, device="cuda")
    mlora.mx4_gemm([y], [mlora.mx4_quantize(x.cuda())], [mlora.MX4Weight.quantize(w.cuda())])
    compare(y, ref.values(*ref.quantize(ref.f64(x))), ref.values(*ref.quantize(ref.f64(w.t()))), F16)


def test_calls_on_two_streams_at_once():
    say("mx4_gemm two streams")
    ws = [operand(n, 2048, 60 + n, 3, mlora.MX4Weight)[0] for n in (264, 4096)]
    xs = [torch.randn((T, 2048), generator=torch.Generator().manual_seed(T)).to(BF16).cuda() for T in (700, 33)]
    want = []
    for x, w in zip(xs, ws):
        y = torch.empty((x.shape[0], w.hout), dtype=BF16, device="cuda")
        mlora.mx4_gemm([y], [mlora.mx4_quantize(x)], [w])
        want.append(y)
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[torch.empty_like(y) for _ in range(8)] for y in want]
    torch.cuda.synchronize()
    for i in range(8):
        for s, x, w, ys in zip(streams, xs, ws, got):
            with torch.cuda.stream(s):
                mlora.mx4_gemm([ys[i]], [mlora.mx4_quantize(x)], [w])
    torch.cuda.synchronize()
    for ys, y in zip(got, want):
        assert all(torch.equal(a, y) for a in ys)


def test_runs_are_alike_on_a_stream_of_ones_own_and_in_a_graph():
    say("mx4_gemm stream and graph")
    T, k, n = 130, 4096, 512
    x = torch.randn((T, k), generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    w, _ = operand(n, k, 4, 3, mlora.MX4Weight)
    y, q = torch.empty((T, n), dtype=BF16, device="cuda"), mlora.mx4_quantize(x)
    mlora.mx4_gemm([y], [q], [w])
    want = y.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = torch.empty_like(y)
        mlora.mx4_gemm([other], [mlora.mx4_quantize(x)], [w])
    s.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mlora.mx4_gemm([y], [mlora.mx4_quantize(x, out=q)], [w])
    for i in range(4):
        x.copy_(torch.randn((T, k), generator=torch.Generator().manual_seed(20 + i)).to(BF16))
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        mlora.mx4_gemm([other], [mlora.mx4_quantize(x)], [w])
        torch.cuda.synchronize()
        assert torch.equal(got, other)
