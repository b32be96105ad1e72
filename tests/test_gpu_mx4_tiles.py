"""mx4_gemm's forms for many tokens, each named before its test runs: blocks that are NaN or far apart, several projections, ends of tiles, few steps."""
import ctypes as C

import numpy as np
import pytest
import torch

import mlora
import mx4_ref as ref
from gpu_common import say
from mlora import _ext
from step_ref import HALF, TINY

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
# one size of every form: of the largest, halves of tiles alone, whole tiles alone, both
ONE = [((64, 64), 201, 2184, 2056), ((128, 64), 300, 1160, 4104), ((128, 128), 1030, 1032, 2056), ((256, 256), 1030, 1160, 4104), ((256, 256), 1030, 392, 12296), ((256, 256), 2570, 1160, 8200)]


def form_of(T, sizes):
    shape, n = (C.c_int32 * 2)(), len(sizes)
    assert _ext.lib().mlora_mx4_form(n, (C.c_int32 * n)(*[k for k, _ in sizes]), (C.c_int32 * n)(*[h for _, h in sizes]), T, shape) == 0
    return tuple(shape)


def operand(rows, k, seed, spread=3, nan=()):
    """A packed operand of random codes, blocks `nan` (row, block) of it NaN, and its values in 64 bits on the device (NaN as zeros)."""
    rng = np.random.default_rng(seed)
    codes, scales = rng.integers(0, 16, (rows, k)), rng.integers(125 - spread, 126, (rows, -(-k // 32))).astype(np.uint8)
    for r, b in nan:
        scales[r, b] = 255
    packed = mlora.MX4Tensor(torch.from_numpy(ref.packed_codes(codes)).cuda(), torch.from_numpy(scales).cuda())
    return packed, torch.from_numpy(np.nan_to_num(ref.values(codes, scales))).cuda()


def compare(y, xv, wv, form, y0=None, rows=None, what=""):
    """The sum of a block's 32 products is exact (multiples of a quarter step, at most 1152 steps).  An instruction brings its block sums and what it adds
    them to to one exponent, that of the largest product or sum among them, and cuts each of them, and their sum, off below 2^-23 of that: of 16 x 16 x 128
    six cuts for 128 columns, of 32 x 32 x 64 two times four.  All of these are at most the sum of the products' magnitudes.  Partial sums of eight wavefronts (of
    two groups of them with 64 x 64) are added in fp32, and y0; the result is rounded to its type once."""
    slim = form in ((16, 16), (32, 16), (16, 32), (32, 32), (32, 64))
    cuts = (6 if slim else 8) * -(-xv.shape[1] // 128) + (7 if slim else form == (64, 64)) + (y0 is not None)
    want, mag = xv @ wv.T, xv.abs() @ wv.abs().T
    if y0 is not None:
        want, mag = want + y0, mag + y0.abs()
    bound = cuts * 2.0 ** -23 * mag
    bound = bound + HALF[y.dtype] * (want.abs() + bound) + TINY[y.dtype]
    bad = (y.double() - want).abs() > bound
    if rows is not None:
        bad &= rows
    at = bad.nonzero()
    assert len(at) == 0, f"{what}: {len(at)} of {bad.numel()} outside, the first at {at[0].tolist()}: {y[tuple(at[0])]} for {want[tuple(at[0])]} +- {bound[tuple(at[0])]}"


def run(T, sizes, form, dtype, accumulate=False, seed=0, spread=3, nan_x=(), nan_w=()):
    what = f"mx4_gemm {form} T={T} {sizes} {dtype} acc={accumulate} spread={spread}"
    say(what)
    assert form_of(T, sizes) == form
    xs = {k: operand(T, k, seed + k, spread, nan_x) for k in {k for k, _ in sizes}}
    ws = [operand(n, k, seed + 17 * i + 1, spread, nan_w) for i, (k, n) in enumerate(sizes)]
    ys = [torch.randn((T, n), device="cuda", generator=torch.Generator("cuda").manual_seed(seed + n)).to(dtype) for _, n in sizes]
    y0s = [y.double() if accumulate else None for y in ys]
    mlora.mx4_gemm(ys, [xs[k][0] for k, _ in sizes], [w for w, _ in ws], accumulate=accumulate)
    for y, y0, (k, n), (_, wv) in zip(ys, y0s, sizes, ws):
        nan = torch.zeros((T, n), dtype=torch.bool, device="cuda")
        nan[[r for r, _ in nan_x]] = True
        nan[:, [r for r, _ in nan_w]] = True
        assert torch.equal(torch.isnan(y), nan), f"{what}: NaN elsewhere than in their rows and columns"
        compare(y, xs[k][1], wv, form, y0, ~nan, what)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("form, T, k, n", ONE)
def test_blocks_far_apart(form, T, k, n, accumulate):
    run(T, [(k, n)], form, BF16, accumulate, spread=40)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("form, T, k, n", ONE)
def test_nan_stays_in_its_row_and_column(form, T, k, n, accumulate):
    """In the first, a middle and the last block, which is short; of the first and last rows, of rows beside tiles' borders and of one in the last tile."""
    last = -(-k // 32) - 1
    rows = [(0, 0), (15, last), (64, last // 2), (127, 5), (128, 1), (T - 1, last)]
    run(T, [(k, n)], form, F16, accumulate, nan_x=rows, nan_w=[(0, last), (17, 0), (255, last // 2), (256, 3), (n - 9, 2), (n - 1, last)])


# Three projections share inputs of two widths; of the 256 x 256 ones, the border between whole tiles and halves is inside the second
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("form, T, sizes", [
    ((128, 64), 300, [(1032, 1032), (520, 2056), (1032, 264)]), ((128, 128), 513, [(1032, 1032), (520, 2056), (1032, 264)]), ((128, 128), 449, [(2184, 2056), (2184, 4104)]),
    ((128, 128), 1030, [(136, 2056), (136, 2056), (136, 2056)]), ((256, 256), 449, [(1160, 4104), (648, 8200), (1160, 264)]),
    ((256, 256), 1721, [(1160, 4104), (648, 8200)]), ((256, 256), 2575, [(1160, 1032), (1160, 6152), (136, 264)]), ((256, 256), 2453, [(1160, 2056), (648, 4104), (1160, 2056)])])
def test_projections_of_one_call(form, T, sizes, accumulate):
    run(T, sizes, form, BF16, accumulate)


@pytest.mark.parametrize("form, k, n, tokens", [
    ((64, 64), 2184, 2056, (193, 255, 256, 257, 319, 320, 321, 447, 448)), ((128, 64), 136, 4104, (129, 191, 192, 193, 255, 256, 257, 321)),
    ((128, 128), 136, 4104, (511, 512, 513, 576, 639, 640, 641, 769, 896)), ((256, 256), 136, 4104, (1023, 1024, 1025, 1088, 1151, 1152, 1153, 1279, 1280, 1281, 1408, 1409))])
def test_tokens_at_the_ends_of_tiles(form, k, n, tokens):
    for T in tokens:
        run(T, [(k, n)], form, F16, seed=T)


@pytest.mark.parametrize("form, T, n", [((128, 64), 300, 4104), ((128, 128), 1030, 2056), ((256, 256), 1030, 4104), ((256, 256), 1030, 12296)])
def test_few_steps(form, T, n):
    """One step to nine of a ring of four stages: the last two are halves of 256 x 256 tiles, and whole ones."""
    for k in (8, 128, 136, 256, 384, 512, 520, 640, 768, 896, 1024, 1032):
        run(T, [(k, n)], form, BF16, seed=k)


@pytest.mark.parametrize("k", [1160, 1280, 1536, 1544, 1672, 1920, 2048, 2056, 2184, 2312, 2560, 2568, 4096, 4104])
def test_steps_of_two_groups(k):
    """The quads of K tiles in halves: of odd and even numbers of them, the last one with one to four tiles, the last tile short."""
    run(201, [(k, 2056)], (64, 64), BF16, seed=k)
    run(201, [(k, 2056)], (64, 64), F16, accumulate=True, seed=k, nan_x=[(200, -(-k // 32) - 1)], nan_w=[(2055, -(-k // 32) - 1)])
