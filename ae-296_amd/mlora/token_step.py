"""One decode step of the attention blocks: 4-bit base projections, every token's adapter, rotation and append, attention.

    step = TokenStep(pool, cache, weights, n_q_heads, rope)
    step.begin(batch, tok_adapter)                  # once per step: both plans
    for layer in range(L):
        a = step.layer(layer, x)                    # [T, Hq, D], what the output projection reads
        ...

The step allocates nothing after its first batch of a size, apart from what the calls take from torch's allocator for their own
length, so it may be captured in a HIP graph once it has run eagerly.  Batches of up to 2^k tokens share one set of buffers: a graph's
replay and other work of the same step object are ordered on one stream.
"""
from __future__ import annotations

from typing import Dict, Optional, Sequence

import torch

from . import ops
from .attention import KVBatch, KVCache, RopeTable, kv_append, plan_attention, prefix_attention
from .pool import AdapterPool
from .w4 import W4Weight, w4_gemv


class TokenStep:
    """`weights[layer][name]` are the base projections of q, k and v (`names`, in that order) as ``W4Weight``; None leaves them
    to the caller, whose base products ``layer`` then takes as `qkv`, or without any the deltas alone are q, k and v."""

    def __init__(self, pool: AdapterPool, cache: KVCache, weights: Optional[Sequence[Dict[str, W4Weight]]], n_q_heads: int,
                 rope: Optional[RopeTable] = None, names: Sequence[str] = ("q", "k", "v")):
        if len(names) != 3:
            raise ValueError("names must be the projections of q, k and v")
        D = cache.head_dim
        self.widths = [n_q_heads * D, cache.n_kv_heads * D, cache.n_kv_heads * D]
        hin = pool.projections[names[0]][0]
        for name, width in zip(names, self.widths):
            if tuple(pool.projections[name]) != (hin, width):
                raise ValueError(f"projection {name} must be {hin} -> {width} in the pool")
        if pool.dtype != cache.dtype or pool.n_layers != cache.n_layers:
            raise ValueError("the pool and the cache must have one dtype and number of layers")
        if weights is not None and len(weights) != pool.n_layers:
            raise ValueError("weights must list every layer")
        for layer in weights or ():
            for name, width in zip(names, self.widths):
                if (layer[name].hin, layer[name].hout) != (hin, width):
                    raise ValueError(f"the 4-bit weight of {name} must be {hin} -> {width}")
        self.pool, self.cache, self.weights, self.n_q_heads, self.rope, self.names = pool, cache, weights, n_q_heads, rope, list(names)
        self.batch: Optional[KVBatch] = None
        self.tok_adapter = None
        # Batch size -> plans and views, power of two -> buffers.  None is ever given back: a graph that was captured with them goes on
        # using them.  Buffers for every size would add up: to 4 GB over the sizes to 512, with four rows of 8 KB a token.
        self._kept, self._buffers = {}, {}
        self._outgrown = []
        self.bad = torch.zeros(1, dtype=torch.int32, device=cache.device)      # tokens that kv_append left out since begin, added up over the layers

    def begin(self, batch: KVBatch, tok_adapter: torch.Tensor) -> None:
        """A step's batch: its tokens, pages and prefixes, and the adapter slot of every token (int32, negative: none).  After a batch that
        was refused ``layer`` raises until the next ``begin``."""
        self.batch = None            # until all of it is accepted: after a refusal the kept plans may be those of two batches
        if tok_adapter.numel() != batch.T:
            raise ValueError("tok_adapter must have one entry for every token of the batch")
        T, n_prefix = batch.T, 0 if batch.prefix_len is None else batch.prefix_len.numel()
        kept = self._kept.get(T)
        if kept is None:
            room = max(1, 1 << (T - 1).bit_length()) if T else 1
            if room not in self._buffers:
                new = dict(dtype=self.cache.dtype, device=self.cache.device)
                self._buffers[room] = [torch.empty((room, w), **new) for w in self.widths] + [torch.empty((room, self.n_q_heads, self.cache.head_dim), **new)]
            *qkv, out = (b[:T] for b in self._buffers[room])
            kept = self._kept[T] = [None, None, qkv, out, -1]
        if n_prefix > kept[4]:            # room for twice as many, so that a growing number of prompts moves the plan a few times only
            holds = n_prefix if kept[1] is None else min(2 * n_prefix, 4096)
            plan = plan_attention(batch, self.cache, self.n_q_heads, room=holds)
            if kept[1] is not None:
                self._outgrown.append(kept[1])
            kept[1], kept[4] = plan, holds        # only now: a batch that was refused must not count as room
        else:
            plan_attention(batch, self.cache, self.n_q_heads, out=kept[1])
        if kept[0] is None:
            kept[0] = ops.plan_decode(tok_adapter, self.pool, n_proj=3)
        else:
            ops.plan_decode(tok_adapter, self.pool, out=kept[0])
        self.bad.zero_()
        kept[3].zero_()              # rows without a request: the attention leaves them alone, and other batches share the buffer
        self.decode_plan, self.attn_plan, self.qkv, self.out = kept[:4]
        self.batch, self.tok_adapter = batch, tok_adapter

    def layer(self, layer: int, x: torch.Tensor, qkv: Optional[Sequence[torch.Tensor]] = None, scale: Optional[float] = None) -> torch.Tensor:
        """Attention output [T, Hq, D] of one layer for its input x [T, hin]; the buffer is the step's own and holds it until the next
        call; rows without a request are zeros.  q, k and v are left in `self.qkv` (or `qkv`), q rotated.  A token whose page or position no table
        holds is counted in `self.bad` (int32, on the device; every layer counts it again): its key is missing and its q not rotated."""
        if self.batch is None:
            raise RuntimeError("begin() names the step's batch first")
        if qkv is not None and self.weights is not None:
            raise ValueError("qkv is for a step without weights of its own")
        ys = list(qkv) if qkv is not None else self.qkv
        if self.weights is not None:
            w4_gemv(ys, [x] * 3, [self.weights[layer][n] for n in self.names])
        ops.bgmv(ys, [x] * 3, self.pool, layer, self.names, self.tok_adapter, plan=self.decode_plan,
                 accumulate=qkv is not None or self.weights is not None)
        D, T = self.cache.head_dim, self.batch.T
        q, k, v = (y.view(T, w // D, D) for y, w in zip(ys, self.widths))
        kv_append(q, k, v, self.cache, layer, self.batch, self.rope, bad=self.bad)
        return prefix_attention(q, self.cache, layer, self.attn_plan, scale=scale, out=self.out)
