"""Keys, values and attention of the tokens whose q, k and v ``bgmv`` / ``sgmv_multi`` have just finished: rotation and append to a
paged cache, and attention in which the keys of a prompt that several requests share are read once for all of them.

In a multi-LoRA batch the requests of one adapter usually start with that adapter's task prompt, so a batch has several
prefixes.  A prefix is written as any request's keys are (a batch whose page table is the prefix's own) and then named by the requests
that follow it: ``KVBatch.req_prefix``.  Every function launches on ``torch.cuda.current_stream()`` and does not synchronise.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional

import torch

from . import _ext

HEAD_DIMS = (64, 128)


class KVCache:
    """Paged keys and values resident in HBM: k and v [n_layers, n_pages, n_kv_heads, page_tokens, head_dim].  Pages are handed
    out by ``allocate`` and taken back by ``release``; the same page ids serve every layer."""

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, page_tokens: int = 16,
                 dtype: torch.dtype = torch.float16, device: str | torch.device = "cuda"):
        if page_tokens < 16 or page_tokens > 256 or page_tokens & (page_tokens - 1):
            raise ValueError("page_tokens must be a power of two in 16..256")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
        if n_layers < 1 or n_pages < 1 or n_kv_heads < 1:
            raise ValueError("n_layers, n_pages and n_kv_heads must be positive")
        self.dtype_code = _ext.dtype_code(dtype)
        self.n_layers, self.n_pages, self.n_kv_heads, self.head_dim, self.page_tokens = n_layers, n_pages, n_kv_heads, head_dim, page_tokens
        self.dtype = dtype
        self.device = torch.device(device)
        shape = (n_layers, n_pages, n_kv_heads, page_tokens, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=self.device)
        self.v = torch.empty(shape, dtype=dtype, device=self.device)
        self._free = list(range(n_pages - 1, -1, -1))
        self._used = set()

    def allocate(self, n: int) -> List[int]:
        """n free page ids."""
        if n < 0 or n > len(self._free):
            raise MemoryError(f"cache full: {n} pages needed, {len(self._free)} free")
        got = [self._free.pop() for _ in range(n)]
        self._used.update(got)
        return got

    def release(self, pages) -> None:
        """Give pages back; what a launch still queued reads of them must be ordered before what overwrites them."""
        pages = [int(p) for p in pages]
        if len(set(pages)) != len(pages) or not self._used.issuperset(pages):
            raise ValueError("release takes pages that allocate gave out, each once")
        self._used.difference_update(pages)
        self._free.extend(reversed(pages))

    @property
    def free_pages(self) -> int:
        return len(self._free)


@dataclass
class KVBatch:
    """The tokens of a step, int32 on the device: token t is position tok_pos[t] of request tok_req[t] (negative: a row without
    a request, left alone everywhere).  Request r follows prefix req_prefix[r] (negative: none) of prefix_len[...] tokens; its
    own keys lie on pages[r], those of prefix f on prefix_pages[f] (-1 behind a list's end)."""
    tok_req: torch.Tensor                          # [T]
    tok_pos: torch.Tensor                          # [T]
    pages: torch.Tensor                            # [n_req, max_pages]
    req_prefix: Optional[torch.Tensor] = None      # [n_req]
    prefix_pages: Optional[torch.Tensor] = None    # [n_prefix, max_prefix_pages]; needed by the attention only
    prefix_len: Optional[torch.Tensor] = None      # [n_prefix]

    @property
    def T(self) -> int:
        return self.tok_req.numel()


class RopeTable:
    """Cosines and sines of every position, float32 [n_pos, rot] (cosines first), from angles in float64: position * frequency
    of pair i, by default base ** (-2 i / rot).  The first `rot` elements of a head turn, pair (i, i + rot / 2) or, interleaved,
    (2 i, 2 i + 1)."""

    def __init__(self, n_pos: int, rot: int, base: float = 10000.0, interleaved: bool = False,
                 frequencies: Optional[torch.Tensor] = None, device: str | torch.device = "cuda"):
        if n_pos < 1 or rot < 16 or rot % 16 or rot > max(HEAD_DIMS):
            raise ValueError("n_pos must be positive and rot a multiple of 16 up to the head's size")
        f = frequencies
        if f is None:
            f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
        if f.numel() != rot // 2:
            raise ValueError(f"frequencies must hold {rot // 2} values")
        angle = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * f.to(device=device, dtype=torch.float64).view(1, -1)
        self.cos_sin = torch.cat((torch.cos(angle), torch.sin(angle)), 1).float()
        self.n_pos, self.rot, self.interleaved = n_pos, rot, interleaved


def kv_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, cache: KVCache, layer: int, batch: KVBatch,
              rope: Optional[RopeTable], q_out: Optional[torch.Tensor] = None, bad: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotate q [T, Hq, D] and k [T, Hkv, D] by their tokens' positions and place k and v on their pages, in one launch;
    returns the rotated q (`q_out`, or q itself in place).  The tokens' rows may be apart (views of one fused projection output).
    ``rope=None`` places k and v as they are.  A token with a request whose position no table holds is left out as a whole and counted in `bad`
    (int32, one value).  `q_out` may be q itself and otherwise overlaps neither q, k nor v; two tokens at one position of one request leave a mixture
    of both there."""
    rc = _ext.host().kv_append(q, k, v, q_out, cache, layer, batch, rope, bad)
    if rc:
        _ext.check(rc)
    return q if q_out is None else q_out


@dataclass
class AttnPlan:
    """Division of one step's attention work, for every layer (written by ``mlora_attn_plan``)."""
    batch: KVBatch
    T: int
    n_q_heads: int
    n_kv_heads: int
    page_tokens: int
    buf: torch.Tensor
    n_req: int = 0
    n_prefix: int = 0


def plan_attention(batch: KVBatch, cache: KVCache, n_q_heads: int, out: Optional[AttnPlan] = None, room: int = 0) -> AttnPlan:
    """Divide the step's attention work once; the plan serves every layer's ``prefix_attention``.  Pass `out` to reuse a plan's
    buffer (no allocation; safe under graph capture; a batch larger than the one it was made for is refused); `room`: prefixes that
    a new buffer is sized for where that is more than the batch has."""
    if n_q_heads < 1 or n_q_heads % cache.n_kv_heads:
        raise ValueError(f"n_q_heads must be a multiple of the cache's {cache.n_kv_heads} key heads")
    n_prefix = 0 if batch.prefix_len is None else batch.prefix_len.numel()
    if out is None:
        need = _ext.lib().mlora_attn_plan_bytes(batch.T, max(n_prefix, room), n_q_heads, cache.n_kv_heads)
        if need < 0:
            _ext.check(need)
        buf = torch.empty(need, dtype=torch.uint8, device=batch.tok_req.device)
    else:
        buf = out.buf
    rc = _ext.host().attn_plan(batch, buf, cache.page_tokens, n_q_heads, cache.n_kv_heads, cache.head_dim)
    if rc:
        _ext.check(rc)
    if out is None:
        return AttnPlan(batch, batch.T, n_q_heads, cache.n_kv_heads, cache.page_tokens, buf, batch.pages.shape[0], n_prefix)
    # only now: a batch that the buffer does not hold was refused and must not be taken for the plan's own
    out.batch, out.T, out.n_q_heads, out.n_kv_heads, out.page_tokens = batch, batch.T, n_q_heads, cache.n_kv_heads, cache.page_tokens
    out.n_req, out.n_prefix = batch.pages.shape[0], n_prefix
    return out


def prefix_attention(q: torch.Tensor, cache: KVCache, layer: int, plan: AttnPlan, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t, h] = softmax(scale * q[t, h] . K) V over positions 0 .. tok_pos[t] of token t's request, its prefix's among them;
    q and out [T, Hq, D] (rows may be apart), scale 1 / sqrt(D) by default (0, or 2^-126 to 2^127 of either sign); out must not overlap q.  A row that sees no key is zeros (one whose
    scores are all minus infinity is NaN, as the softmax is); rows without a request keep what `out` held (zeros in a new one)."""
    if out is None:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    if scale is None:
        scale = cache.head_dim ** -0.5
    rc = _ext.host().prefix_attention(q, out, cache, layer, plan, float(scale))
    if rc:
        _ext.check(rc)
    return out
