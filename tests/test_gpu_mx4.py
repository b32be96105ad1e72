"""Microscaled 4-bit quantisation against the definition, bit for bit."""
import numpy as np
import pytest
import torch

import mlora
import mx4_ref as ref
from gpu_common import say

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def quantized(x):
    """(values that the kernel's operand stands for, values by the definition), as 64-bit arrays."""
    q = mlora.mx4_quantize(x)
    got = ref.f64(q.values(x.dtype))
    return got, ref.values(*ref.quantize(ref.f64(x)))


def same(got, want):
    assert got.shape == want.shape
    bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), f"{int(bad.sum())} of {bad.size}, first at {tuple(np.argwhere(bad)[0])}: got {got[bad][0]!r}, want {want[bad][0]!r}"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows, k", [(1, 8), (1, 32), (2, 40), (3, 4096), (15, 128), (16, 512), (17, 520), (33, 1000), (64, 2752), (129, 136)])
def test_values_of_sizes(rows, k, dtype):
    say(f"mx4 quantize {rows}x{k} {dtype}")
    g = torch.Generator().manual_seed(rows * 7 + k)
    x = (torch.randn((rows, k), generator=g) * torch.exp2(torch.randint(-6, 6, (rows, 1), generator=g).float())).to(dtype).cuda()
    same(*quantized(x))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_every_finite_number_under_every_larger_one(dtype):
    """Each 16-bit pattern beside a largest element that puts the block's power of two where the pattern rounds: ties, subnormals, both signs."""
    say(f"mx4 all patterns {dtype}")
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    bits = bits[torch.isfinite(bits)]
    for shift in (0, 1, 2, 3):
        x = torch.zeros((len(bits), 32), dtype=dtype)
        x[:, 5] = bits
        x[:, 31] = (bits.double().abs() * 2.0 ** shift * 1.25).clamp(max=torch.finfo(dtype).max).to(dtype)
        same(*quantized(x.cuda()))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_infinities_and_nan_make_their_block_nan(dtype):
    say(f"mx4 not finite {dtype}")
    x = torch.randn((20, 200), generator=torch.Generator().manual_seed(1)).to(dtype)
    x[3, 40], x[5, 199], x[19, 0], x[7, 64:96] = float("inf"), float("nan"), float("-inf"), float("nan")
    x[9] = 0
    x[10] = -0.0
    got, want = quantized(x.cuda())
    assert np.isnan(got[3, 32:64]).all() and np.isnan(got[5, 192:]).all() and np.isfinite(got[3, :32]).all()
    same(got, want)


def test_codes_and_scales_are_the_definitions():
    """The operand itself, and its sign of zero, by the packed layout that the header describes; columns past the last are zero codes."""
    rows, k = 19, 712
    x = torch.randn((rows, k), generator=torch.Generator().manual_seed(2)).to(BF16)
    x[4, :32] = 0
    x[4, 3] = -0.0
    say("mx4 layout")
    q = mlora.mx4_quantize(x.cuda())
    p = q.packed.cpu().numpy()
    codes, scales = ref.quantize(ref.f64(x))
    tiles, quads = -(-k // 128), -(-k // 512)
    plane = p[:2 * tiles * 1024].reshape(2, tiles, 4, 16, 16)
    exps = p[2 * tiles * 1024:].reshape(2, quads, 4, 16, 4)
    for r in range(rows):
        for b in range(tiles * 4):
            got = plane[r // 16, b // 4, b % 4, r % 16]
            want = np.zeros(32, int)
            part = codes[r, 32 * b:32 * b + 32]
            want[:len(part)] = part
            assert np.array_equal(got, ref.packed_codes(want[None])[0]), (r, b)
            assert exps[r // 16, b // 16, b % 4, r % 16, b // 4 % 4] == (scales[r, b] if b < scales.shape[1] else 0), (r, b)


@pytest.mark.parametrize("rows, k", [(1, 8), (5, 72), (16, 128), (40, 1040)])
def test_packed_from_a_checkpoint(rows, k):
    say(f"mx4 pack {rows}x{k}")
    rng = np.random.default_rng(rows + k)
    codes = rng.integers(0, 16, (rows, k))
    scales = rng.integers(0, 256, (rows, -(-k // 32))).astype(np.uint8)
    t = mlora.MX4Tensor(torch.from_numpy(ref.packed_codes(codes)).cuda(), torch.from_numpy(scales).cuda())
    with np.errstate(over="ignore"):
        want = torch.from_numpy(ref.values(codes, scales))
        same(ref.f64(t.values(BF16)), ref.f64(want.to(torch.float32).to(BF16)))
        same(ref.f64(t.values(F16)), ref.f64(want.to(torch.float32).to(F16)))


def test_rows_apart_and_reused_buffers():
    say("mx4 strides")
    base = torch.randn((40, 600), generator=torch.Generator().manual_seed(4)).to(F16).cuda()
    x = base[:, 8:208]
    q = mlora.mx4_quantize(x)
    same(ref.f64(q.values(F16)), ref.values(*ref.quantize(ref.f64(x))))
    again = mlora.mx4_quantize(base[:3, 16:24], out=q)
    assert again is q and (q.rows, q.k) == (3, 8)
    same(ref.f64(q.values(F16)), ref.values(*ref.quantize(ref.f64(base[:3, 16:24]))))
    out = torch.full((3, 64), 7.0, dtype=F16, device="cuda")
    q.values(out=out[:, 16:24])
    assert (out[:, :16] == 7).all() and (out[:, 24:] == 7).all()
    same(ref.f64(out[:, 16:24]), ref.values(*ref.quantize(ref.f64(base[:3, 16:24]))))


def test_a_weight_is_quantised_along_its_input():
    say("mx4 weight")
    w = torch.randn((264, 48), generator=torch.Generator().manual_seed(5)).to(BF16).cuda()
    m = mlora.MX4Weight.quantize(w)
    assert (m.hin, m.hout) == (264, 48)
    same(ref.f64(m.values(BF16)), ref.values(*ref.quantize(ref.f64(w.t()))))


def test_refusals_on_the_device():
    say("mx4 refusals")
    x = torch.zeros((4, 64), dtype=F16, device="cuda")
    q = mlora.mx4_quantize(x)
    for bad in (x[:, :12], x[:, 4:]):                              # a width, and an address
        with pytest.raises(mlora.MloraError):
            mlora.mx4_quantize(bad)
    for bad in (x.t(), x[0], x.unsqueeze(0)):
        with pytest.raises(ValueError):
            mlora.mx4_quantize(bad)
    with pytest.raises(TypeError):
        mlora.mx4_quantize(x.float())
    with pytest.raises(mlora.MloraError):
        mlora.mx4_quantize(torch.zeros((40, 64), dtype=F16, device="cuda"), out=q)
    assert (q.rows, q.k) == (4, 64)                                # what it was
    with pytest.raises(TypeError):
        q.values(torch.float32)
    with pytest.raises(ValueError):
        q.values(out=x[:3])
    w, y = mlora.MX4Weight.quantize(torch.zeros((64, 16), dtype=F16, device="cuda")), torch.zeros((4, 16), dtype=F16, device="cuda")
    for ys, xs, ws in (([y, y], [q], [w]), ([y[:3]], [q], [w]), ([y[:, :8]], [q], [w]), ([y], [mlora.mx4_quantize(x[:, :32])], [w]), ([y] * 9, [q] * 9, [w] * 9)):
        with pytest.raises(ValueError):
            mlora.mx4_gemm(ys, xs, ws)
    with pytest.raises(TypeError):
        mlora.mx4_gemm([y.float()], [q], [w])
    with pytest.raises(TypeError):
        mlora.mx4_gemm([y, y.bfloat16()], [q, q], [w, w])
    with pytest.raises(mlora.MloraError):
        mlora.mx4_gemm([y, y], [q, q], [w, w])                     # one y twice


def test_no_rows():
    say("mx4 no rows")
    q = mlora.mx4_quantize(torch.empty((0, 64), dtype=F16, device="cuda"))
    assert q.values(F16).shape == (0, 64)
    y = torch.empty((0, 16), dtype=F16, device="cuda")
    mlora.mx4_gemm([y], [q], [mlora.MX4Weight.quantize(torch.ones((64, 16), dtype=F16, device="cuda"))])
