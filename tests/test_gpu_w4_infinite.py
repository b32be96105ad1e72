"""4-bit products of rows that hold infinities, NaN or values whose products with 16 + c leave fp32: what the formula gives in 64 bits, and the
rows beside them what they are without such a row."""
import numpy as np
import pytest
import torch

import mlora
from gpu_common import say
from step_ref import check, f64, store_bound, w4_exact
from test_gpu_w4 import weight

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


def definition(x, codes, scales, zeros, group, y0):
    """sum_k s (c - z) x_k in 64 bits, 0 * infinity being NaN."""
    s, c = f64(scales), f64(codes)
    rows = np.arange(c.shape[0]) // group
    with np.errstate(invalid="ignore"):
        terms = f64(x)[:, None] * ((c - (8.0 if zeros is None else f64(zeros)[rows])) * s[rows])
        return terms.sum(0) + (0.0 if y0 is None else f64(y0))


def same_or_close(got, want, dtype, what):
    got = f64(got)
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    assert np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)]), f"{what}: infinities of another sign"
    check(torch.from_numpy(np.where(odd, 0.0, got)), np.where(odd, 0.0, want), store_bound(np.where(odd, 0.0, want), dtype) * (1 + 2.0 ** -20), what)


# sizes of every shape of workgroup on a device of 256 compute units; a column's last tile is whole or not
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group, zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("T, hin, hout", [(1, 520, 72), (5, 1024, 4104), (17, 904, 72), (20, 520, 4104), (40, 776, 4104), (320, 640, 8192),
                                          (60, 392, 16400), (190, 264, 16400)])
def test_rows_with_infinities(T, hin, hout, group, zeros, dtype):
    say(f"w4 infinities T={T} {hin}->{hout} group={group} zeros={zeros} {dtype}")
    accumulate = hout % 16 != 0
    codes, scales, z = weight(hin, hout, group, zeros, dtype, T)
    w = mlora.W4Weight(codes, scales, z, group=group)
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn((T, hin), device="cuda", generator=g).to(dtype)
    y0 = torch.randn((T, hout), device="cuda", generator=g).to(dtype)
    plain = y0.clone()
    mlora.w4_gemv([plain], [x], [w], accumulate=accumulate)
    rows = {0: {hin // 2: INF}}
    if T > 3:
        rows[T - 1] = {hin - 1: -INF}
        rows[T // 2] = {0: INF, hin // 3: -INF}
        rows[T // 3] = {hin - 8: NAN}
    for t, at in rows.items():
        for k, v in at.items():
            x[t, k] = v
    y = y0.clone()
    mlora.w4_gemv([y], [x], [w], accumulate=accumulate)
    for t in rows:
        same_or_close(y[t], definition(x[t], codes, scales, z, group, y0[t] if accumulate else None), dtype, f"row {t}")
        y[t] = plain[t]
    assert torch.equal(y, plain), "rows beside an infinite one"


@pytest.mark.parametrize("group, zeros", [(32, False), (128, True)])
@pytest.mark.parametrize("T, hin, hout", [(2, 520, 72), (5, 264, 4104), (40, 776, 4104), (60, 392, 16400), (190, 264, 16400)])
def test_large_finite_values(T, hin, hout, group, zeros):
    """2^125 among values near one: 31 times it is beyond fp32, its products with (c - z) s are not beyond bf16."""
    say(f"w4 2^125 T={T} {hin}->{hout} group={group}")
    codes, scales, z = weight(hin, hout, group, zeros, BF16, 3 * T)
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn((T, hin), device="cuda", generator=g).to(BF16)
    x[0, 17] = 2.0 ** 125
    x[T - 1, hin - 1] = -2.0 ** 125
    y = torch.empty((T, hout), device="cuda", dtype=BF16)
    mlora.w4_gemv([y], [x], [mlora.W4Weight(codes, scales, z, group=group)])
    for t in (0, T - 1):
        want = definition(x[t], codes, scales, z, group, None)
        # what the fast sum gave stays where it was finite: sums of 31 |x| in fp32
        _, bound = w4_exact(x[t:t + 1], codes, scales, z, group)
        assert np.isfinite(want).all()
        check(y[t], want, bound[0] + store_bound(np.abs(want) + bound[0], BF16), f"row {t}")


def test_infinite_scales_and_sums():
    """A scale of infinity makes its column infinite or NaN; an infinite y stays; nothing of it reaches another column."""
    codes, scales, z = weight(256, 64, 64, True, F16, 1)
    x = torch.randn((3, 256), device="cuda").to(F16)
    y0 = torch.randn((3, 64), device="cuda").to(F16)
    plain = y0.clone()
    mlora.w4_gemv([plain], [x], [mlora.W4Weight(codes, scales, z, group=64)], accumulate=True)
    scales[2, 5] = INF
    y = y0.clone()
    y[1, 9] = -INF
    mlora.w4_gemv([y], [x], [mlora.W4Weight(codes, scales, z, group=64)], accumulate=True)
    for t in range(3):
        want = definition(x[t], codes, scales, z, 64, y0[t])
        assert not torch.isfinite(y[t, 5]) and not np.isfinite(want[5])
    assert y[1, 9] == -INF
    y[:, 5], y[1, 9] = plain[:, 5], plain[1, 9]
    assert torch.equal(y, plain)
