"""Microscaled 4-bit numbers (MXFP4) and base projections on them: weights and inputs both in 4 bits, for prompts as for decode batches.

An element is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, times a power of two that the 32 columns of its block share:

    X = max(floor(log2(max |x| of the block)) - 2, -127),   value = the nearest of the grid to x / 2^X, of two the even code's, times 2^X

so a block's largest magnitude lies in 4 .. 8 steps and saturates above 6.  A block with an infinity or a NaN is NaN as a whole.  ``w4_gemv`` keeps the inputs
in 16 bits and reads a weight again every few tokens; here an input is rounded to 4 bits as well and the product runs on the 4-bit matrix instructions.
Launches go to ``torch.cuda.current_stream()`` and do not synchronise.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _ext

BLOCK = 32


def _packed_bytes(rows: int, k: int) -> int:
    need = _ext.lib().mlora_mx4_bytes(rows, k)
    if need < 0:
        _ext.check(need)
    return need


class MX4Tensor:
    """A packed operand [rows, k]: tokens of an input (``mx4_quantize``) or the output columns of a weight.  From a checkpoint's form:
    codes uint8 [rows, k / 2], an even column in the low half of a byte, and scales uint8 [rows, ceil(k / 32)], 127 + X (255: NaN); the
    sources are copied once and not needed afterwards."""

    __slots__ = ("rows", "k", "packed")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dim() != 2 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes must be uint8 [rows, k / 2] and scales uint8 [rows, ceil(k / 32)]")
        self.rows, self.k = codes.shape[0], 2 * codes.shape[1]
        need = _packed_bytes(self.rows, self.k)
        if tuple(scales.shape) != (self.rows, -(-self.k // BLOCK)):
            raise ValueError(f"scales must be [{self.rows}, {-(-self.k // BLOCK)}]")
        for t in (codes, scales):
            if not t.is_cuda:
                raise ValueError("mlora kernels take device tensors; got a CPU tensor")
            if t.device.index != torch.cuda.current_device():
                raise ValueError("codes and scales must be on the current device")
            if not t.is_contiguous():
                raise ValueError("mlora kernels take contiguous tensors")
        self.packed = torch.empty(need, dtype=torch.uint8, device=codes.device)
        _ext.check(_ext.lib().mlora_mx4_pack(codes.data_ptr(), scales.data_ptr(), self.rows, self.k, self.packed.data_ptr(), need,
                                             _ext.current_stream_ptr()))

    @classmethod
    def empty(cls, rows: int, k: int, device: str | torch.device = "cuda") -> "MX4Tensor":
        """Room for an operand of up to so many rows, for ``mx4_quantize(..., out=)``; until then it holds anything."""
        made = cls.__new__(cls)
        made.packed, made.rows, made.k = torch.empty(_packed_bytes(rows, k), dtype=torch.uint8, device=device), rows, k
        return made

    def values(self, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """What the operand stands for, [rows, k] in a 16-bit type (into `out`, whose rows may be apart): exact for what was quantised from it."""
        got = _ext.host().mx4_values(self, out, _ext.dtype_code(dtype) if out is None else 0)
        if type(got) is int:
            _ext.check(got)
        return got


def mx4_quantize(x: torch.Tensor, out: Optional[MX4Tensor] = None) -> MX4Tensor:
    """A 16-bit tensor [rows, k] (its rows may be apart) in the form above, one launch.  Pass `out` to reuse an operand's buffer, for a batch it was made
    for or a smaller one (no allocation; it is then what is returned)."""
    got = _ext.host().mx4_quantize(x, None if out is None else out.packed)
    if type(got) is int:
        _ext.check(got)
    made = MX4Tensor.__new__(MX4Tensor) if out is None else out
    made.packed, made.rows, made.k = got           # only now: a refused call leaves `out` what it was
    return made


class MX4Weight(MX4Tensor):
    """A weight hin -> hout as ``mx4_gemm`` takes it: codes uint8 [hout, hin / 2] and scales uint8 [hout, ceil(hin / 32)], blocks along the input."""

    __slots__ = ()

    @property
    def hin(self) -> int:
        return self.k

    @property
    def hout(self) -> int:
        return self.rows

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "MX4Weight":
        """From a 16-bit weight [hin, hout] (the layout of ``layer_weight.q_weight_``)."""
        if w.dim() != 2:
            raise ValueError("expected a weight [hin, hout]")
        made = cls.__new__(cls)
        made.packed = None
        return mx4_quantize(w.t().contiguous(), out=made)


def mx4_gemm(ys: Sequence[torch.Tensor], xs: Sequence[MX4Tensor], ws: Sequence[MX4Tensor], accumulate: bool = False) -> None:
    """Base products for up to 8 projections of one layer: ``ys[p] (+)= xs[p] @ ws[p]^T``, xs[p] [T, hin], ws[p] [hout, hin], ys[p] [T, hout] in
    one 16-bit type, no y overlapping another one, an x or a weight; projections of one input take the same xs[p].  ``bgmv`` or ``sgmv_multi`` then add the
    adapters' deltas from the 16-bit input.  Besides the rounding of the result it is off by less than (8 ceil(hin / 128) + 8) 2^-23 of the sum of its products'
    magnitudes: the matrix instruction cuts what it adds off below 2^-23 of the largest, so small blocks beside large ones that cancel are lost."""
    rc = _ext.host().mx4_gemm(ys, xs, ws, accumulate)
    if rc:
        _ext.check(rc)
