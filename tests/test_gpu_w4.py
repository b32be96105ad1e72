"""Base projections on 4-bit weights against the 64-bit product."""
import numpy as np
import pytest
import torch

import mlora
from gpu_common import say
from step_ref import check, store_bound, w4_exact

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def weight(hin, hout, group, zeros, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = -(-hin // group)
    codes = torch.randint(0, 16, (hin, hout), device="cuda", dtype=torch.uint8, generator=g)
    scales = (torch.rand((n, hout), device="cuda", generator=g) * 0.01 + 0.002).to(dtype)
    z = torch.randint(0, 16, (n, hout), device="cuda", dtype=torch.uint8, generator=g) if zeros else None
    return codes, scales, z


def run(T, hin, hout, group, zeros, dtype, seed=0, accumulate=False, mean=0.0):
    say(f"w4 T={T} {hin}->{hout} group={group} zeros={zeros} {dtype} acc={accumulate}")
    codes, scales, z = weight(hin, hout, group, zeros, dtype, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    x = (torch.randn((T, hin), device="cuda", generator=g) + mean).to(dtype)
    y = torch.randn((T, hout), device="cuda", generator=g).to(dtype)
    y0 = y.clone() if accumulate else None
    mlora.w4_gemv([y], [x], [mlora.W4Weight(codes, scales, z, group=group)], accumulate=accumulate)
    want, bound = w4_exact(x, codes, scales, z, group, y0)
    check(y, want, bound + store_bound(np.abs(want) + bound, dtype), f"T={T} {hin}->{hout}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group, zeros", [(32, True), (32, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("T, hin, hout", [(1, 512, 256), (5, 1024, 200), (16, 264, 136), (33, 640, 96)])
def test_product(T, hin, hout, group, zeros, dtype):
    run(T, hin, hout, group, zeros, dtype)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 127, 128, 129, 200])
def test_numbers_of_tokens(T):
    run(T, 384, 144, 64, True, BF16, seed=T)


@pytest.mark.parametrize("hin", [8, 24, 32, 40, 120, 128, 136, 248, 1000, 4096, 11008])
def test_input_widths(hin):
    """The last group and the last tile of a column end anywhere."""
    run(3, hin, 64, 128, True, F16, seed=hin)
    run(18, hin, 64, 32, False, BF16, seed=hin)


@pytest.mark.parametrize("hout", [8, 16, 24, 56, 64, 72, 128, 1032, 4096])
def test_output_widths(hout):
    run(2, 256, hout, 64, False, F16, seed=hout)
    run(40, 256, hout, 32, True, F16, seed=hout)


@pytest.mark.parametrize("group, zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("T, hin, hout", [
    (16, 648, 4104), (1, 1032, 4104),      # two column tiles a workgroup: more than one round of single ones
    (17, 904, 72), (32, 1416, 2048),       # the same in two token blocks
    (20, 520, 4104), (64, 1032, 4096),     # x shared over 32 columns
    (40, 776, 4104), (21, 264, 8200), (130, 2056, 2056),      # over 64
    (300, 1000, 8200), (330, 8, 8192), (300, 136, 8248), (320, 640, 8192),    # at groups of 128 over 128
    (60, 392, 16400), (64, 1016, 16384), (190, 264, 16400)])                  # 64 tokens, over 128 and 256
def test_every_form(T, hin, hout, group, zeros):
    """Sizes on either side of the lines between the kernel's forms, on a device of 256 compute units."""
    run(T, hin, hout, group, zeros, F16 if hout % 16 else BF16, seed=T, accumulate=hin % 16 != 0)


@pytest.mark.parametrize("T", [1, 20, 70])
def test_accumulates(T):
    run(T, 512, 256, 64, True, F16, accumulate=True)


def test_inputs_far_from_zero():
    """A mean of 3 makes the sums that come off at the end as large as they get."""
    run(4, 4096, 128, 128, True, BF16, mean=3.0)
    run(4, 4096, 128, 32, False, F16, mean=3.0)


def test_projections_of_one_call_and_rows_left_alone():
    """Unlike widths, groups and zero points in one call; rows and columns of neighbours stay as they were."""
    shapes = [(256, 512, 64, True), (256, 128, 32, False), (520, 24, 128, True)]
    T = 9
    ws = [weight(*s, F16, 7 + i) for i, s in enumerate(shapes)]
    xs = [torch.randn((T, s[0]), device="cuda").to(F16) for s in shapes]
    whole = [torch.full((T + 2, s[1]), 5.0, device="cuda", dtype=F16) for s in shapes]
    ys = [w[1:T + 1] for w in whole]
    mlora.w4_gemv(ys, xs, [mlora.W4Weight(*w, group=s[2]) for w, s in zip(ws, shapes)])
    for x, y, w, s, all_rows in zip(xs, ys, ws, shapes, whole):
        want, bound = w4_exact(x, *w, s[2])
        check(y, want, bound + store_bound(np.abs(want) + bound, F16))
        assert (all_rows[0] == 5.0).all() and (all_rows[-1] == 5.0).all()


def test_no_tokens():
    w = mlora.W4Weight(*weight(64, 64, 32, False, F16, 0), group=32)
    mlora.w4_gemv([torch.empty((0, 64), device="cuda", dtype=F16)], [torch.empty((0, 64), device="cuda", dtype=F16)], [w])


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantized_weight_is_within_half_a_step(symmetric):
    """The identity as input gives the weights back: each within half a step of its group (and the scale's own rounding to 16 bits)."""
    hin, hout, group = 136, 72, 64
    w = (torch.randn((hin, hout), device="cuda") * 0.1).to(F16)
    codes, scales, zeros = mlora.w4_quantize(w, group, symmetric)
    y = torch.empty((hin, hout), device="cuda", dtype=F16)
    mlora.w4_gemv([y], [torch.eye(hin, device="cuda", dtype=F16)], [mlora.W4Weight.quantize(w, group, symmetric)])
    step = scales.double().repeat_interleave(group, 0)[:hin]
    # the scale is rounded by 2^-11 of itself, at up to 15 steps; the zero point of an asymmetric group by half a step more
    limit = step * ((0.5 if symmetric else 1.0) + 15 * 2.0 ** -11 + 2.0 ** -7)
    assert ((y.double() - w.double()).abs() <= limit).all()
    assert int(codes.max()) <= 15 and (zeros is None) == symmetric


def test_captured_call_replays():
    """Several replays of a captured call with eager work between them; every replay sees the input of its time."""
    codes, scales, z = weight(512, 256, 64, True, F16, 3)
    w = mlora.W4Weight(codes, scales, z, group=64)
    x = torch.randn((7, 512), device="cuda").to(F16)
    y = torch.empty((7, 256), device="cuda", dtype=F16)
    mlora.w4_gemv([y], [x], [w])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mlora.w4_gemv([y], [x], [w])
    for i in range(4):
        x.copy_(torch.randn((7, 512), device="cuda").to(F16))
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        mlora.w4_gemv([y], [x], [w])
        assert torch.equal(got, y)
        want, bound = w4_exact(x, codes, scales, z, 64)
        check(got, want, bound + store_bound(np.abs(want) + bound, F16), f"replay {i}")


def test_calls_on_two_streams():
    codes, scales, z = weight(1024, 512, 128, False, BF16, 5)
    w = mlora.W4Weight(codes, scales, z, group=128)
    xs = [torch.randn((t, 1024), device="cuda").to(BF16) for t in (3, 70)]
    ys = [torch.empty((t, 512), device="cuda", dtype=BF16) for t in (3, 70)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, x, y in zip(streams, xs, ys):
            with torch.cuda.stream(s):
                mlora.w4_gemv([y], [x], [w])
    torch.cuda.synchronize()
    for x, y in zip(xs, ys):
        want, bound = w4_exact(x, codes, scales, z, 128)
        check(y, want, bound + store_bound(np.abs(want) + bound, BF16))
