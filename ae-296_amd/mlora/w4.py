"""Base projections of decode tokens on 4-bit weights: the counterpart of ``gemm_lora``'s base product for the few rows of a
decode batch, whose LoRA deltas ``bgmv`` adds.

    y[t, n] = sum_g scales[g, n] * sum_{k in group g} (codes[k, n] - zeros[g, n]) * x[t, k]

with a scale (and optionally a zero point, 8 otherwise) for every `group` rows of a column.  A row with an infinite or NaN x gives what the
formula gives, but takes longer (32 tokens, 11008 -> 4096: 17 us, 230 with one such row): rows of x that nobody reads should hold numbers.  Launches go to
``torch.cuda.current_stream()`` and do not synchronise.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _ext

GROUPS = (32, 64, 128)


def w4_quantize(w: torch.Tensor, group: int = 128, symmetric: bool = True) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Round-to-nearest 4-bit form of a weight [hin, hout]: (codes uint8 [hin, hout], scales [groups, hout] of w's type,
    zeros uint8 [groups, hout] or None where symmetric).  Symmetric: codes 1..15 around 8, the group's largest magnitude at 7 steps;
    otherwise the group's range (and zero) is spread over 0..15."""
    if w.dim() != 2 or group not in GROUPS:
        raise ValueError(f"expected a weight [hin, hout] and a group in {GROUPS}")
    _ext.dtype_code(w.dtype)
    hin, hout = w.shape
    n = -(-hin // group)
    f = torch.zeros((n * group, hout), dtype=torch.float32, device=w.device)
    f[:hin] = w.float()
    f = f.view(n, group, hout)
    if symmetric:
        scales = (f.abs().amax(1) / 7).to(w.dtype)
        zeros, mid = None, 8.0
    else:
        lo, hi = f.amin(1).clamp(max=0), f.amax(1).clamp(min=0)
        scales = ((hi - lo) / 15).to(w.dtype)
        step = torch.where(scales == 0, torch.ones_like(scales), scales).float()
        zeros = (-lo / step).round().clamp(0, 15).to(torch.uint8)
        mid = zeros.float()[:, None]
    step = torch.where(scales == 0, torch.ones_like(scales), scales).float()[:, None]
    codes = (f / step + mid).round().clamp(1 if symmetric else 0, 15).to(torch.uint8).view(n * group, hout)[:hin]
    return codes.contiguous(), scales, zeros


class W4Weight:
    """A 4-bit weight laid out for ``w4_gemv``: codes uint8 [hin, hout] (one a byte, the low four bits count), scales
    [ceil(hin / group), hout] float16 or bfloat16 (the type of the activations it will meet), zeros uint8 of the scales'
    shape or None.  The sources are copied into `packed` once and not needed afterwards."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, group: int = 128):
        if codes.dim() != 2 or codes.dtype != torch.uint8:
            raise TypeError("codes must be uint8 [hin, hout]")
        if group not in GROUPS:
            raise ValueError(f"group must be one of {GROUPS}")
        self.hin, self.hout = codes.shape
        self.group = group
        self.dtype = scales.dtype
        self.dtype_code = _ext.dtype_code(scales.dtype)
        groups = -(-self.hin // group)
        if tuple(scales.shape) != (groups, self.hout):
            raise ValueError(f"scales must be [{groups}, {self.hout}]")
        if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
            raise ValueError("zeros must be uint8 of the scales' shape")
        self.has_zeros = zeros is not None
        lib = _ext.lib()
        need = lib.mlora_w4_packed_bytes(self.hin, self.hout, group, int(self.has_zeros))
        if need < 0:
            _ext.check(need)
        for t in (codes, scales, zeros):
            if t is None:
                continue
            if not t.is_cuda:
                raise ValueError("mlora kernels take device tensors; got a CPU tensor")
            if t.device != codes.device or t.device.index != torch.cuda.current_device():
                raise ValueError("codes, scales and zeros must be on the current device")
            if not t.is_contiguous():
                raise ValueError("mlora kernels take contiguous tensors")
        self.packed = torch.empty(need, dtype=torch.uint8, device=codes.device)
        _ext.check(lib.mlora_w4_pack(codes.data_ptr(), scales.data_ptr(), _ext.ptr(zeros), self.hin, self.hout, group,
                                     self.packed.data_ptr(), need, _ext.current_stream_ptr()))

    @classmethod
    def quantize(cls, w: torch.Tensor, group: int = 128, symmetric: bool = True) -> "W4Weight":
        """From a 16-bit weight [hin, hout] (the layout of ``layer_weight.q_weight_``), rounded to nearest (``w4_quantize``)."""
        return cls(*w4_quantize(w, group, symmetric), group=group)


def w4_gemv(ys: Sequence[torch.Tensor], xs: Sequence[torch.Tensor], ws: Sequence[W4Weight], accumulate: bool = False) -> None:
    """Base products for up to 8 projections of one layer in one launch: ``ys[p] (+)= xs[p] @ ws[p]``, xs[p] [T, hin], ys[p]
    [T, hout], no y overlapping another one or an x.  Made for decode batches (the weights are read again every 16, 32 or 64 tokens); ``bgmv(ys, xs, ...)`` then adds the
    adapters' deltas."""
    rc = _ext.host().w4_gemv(ys, xs, ws, accumulate)
    if rc:
        _ext.check(rc)
