"""Plain 64-bit forms of the operators around the LoRA apply, and the bounds that their kernels' roundings allow."""
from __future__ import annotations

import numpy as np
import torch

U32 = 2.0 ** -24                                                      # half a step of fp32, relative
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}         # half a step of the 16-bit types
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}       # half of their smallest step


def f64(t):
    return t.detach().cpu().double().numpy()


def store_bound(want, dtype):
    """What one rounding of the result to the 16-bit type may move it by."""
    return HALF[dtype] * np.abs(want) + TINY[dtype]


# ---------------------------------------------------------------- 4-bit weights
def w4_exact(x, codes, scales, zeros, group, y0=None):
    """(result, bound).  The kernel adds 2 * group products of at most 31 |x| per group in fp32, then the groups; every addition is off
    by U32 of a partial sum, which no order makes larger than the sum of the magnitudes."""
    x, c, s = f64(x), f64(codes), f64(scales)
    hin, hout = c.shape
    z = np.full(s.shape, 8.0) if zeros is None else f64(zeros)
    rows = np.arange(hin) // group
    y = x @ ((c - z[rows]) * s[rows])
    mag = np.abs(x) @ (62.0 * np.abs(s[rows]))
    if y0 is not None:
        y = y + f64(y0)
        mag = mag + np.abs(f64(y0))
    return y, (hin + 16) * U32 * mag


# ---------------------------------------------------------------- rotation
def rope_angles(pos, rot, base=10000.0):
    return np.asarray(pos, np.float64)[:, None] * base ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)


def rope_exact(x, pos, rot, interleaved, base=10000.0):
    """(result, bound): cosine, sine, two products and a sum, each off by U32, on values of at most |u| + |w|; the table's angles are
    computed in 64 bits on the device, off by a few steps of 2^-53 of the angle."""
    x = f64(x)
    out, mag = x.copy(), np.zeros_like(x)
    if rot:
        a = rope_angles(pos, rot, base)[:, None]
        c, s = np.cos(a), np.sin(a)
        u, w = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        out[..., u] = x[..., u] * c - x[..., w] * s
        out[..., w] = x[..., u] * s + x[..., w] * c
        mag[..., u] = mag[..., w] = np.abs(x[..., u]) + np.abs(x[..., w])
    far = 1.0 + (np.abs(np.asarray(pos, np.float64)).max(initial=0.0) * 2.0 ** -50) / U32
    return out, (3 + far) * U32 * mag


# ---------------------------------------------------------------- attention
def attention_exact(q, keys, values, scale, dtype):
    """One query row over its visible keys (64-bit arrays): (result, bound).  The bound counts: the fp32 sum of a score's D products and its
    scaling (they move an exponent), the exponential (2 steps), the rounding of a weight to 16 bits (HALF of it, or half of the
    smallest step) in both sums - sum r(p) v / sum r(p) is off by (sum |r(p) - p| |v| + |out| sum |r(p) - p|) / sum r(p), where |out| is at
    most sum p |v| / sum p -, the fp32 sums over n keys in numerator and denominator, and the joining of parts."""
    D = q.shape[0]
    n = keys.shape[0]
    if n == 0:
        return np.zeros(D), np.full(D, TINY[dtype])
    s = keys @ q * scale
    p = np.exp(s - s.max())
    l = p.sum()
    out = p @ values / l
    exponent = ((D + 2) * U32 * np.abs(keys) @ np.abs(q) * abs(scale)).max() + 6 * U32 * np.abs(s).max()
    rel = 2 * np.expm1(exponent) + 2 * 2.0 ** -22 + 2 * HALF[dtype] / (1 - HALF[dtype]) + 2 * (n + 80) * U32
    spread = p @ np.abs(values) / l
    return out, rel * spread + 2 * n * TINY[dtype] * np.abs(values).max(0) / l + HALF[dtype] * np.abs(out) + TINY[dtype]


def check(got, want, bound, what=""):
    got = f64(got)
    bad = ~(np.abs(got - want) <= bound)          # a NaN is bad too
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.size} outside the bound; first at {tuple(np.argwhere(bad)[0])}: "
                           f"got {got[bad][0]!r}, want {want[bad][0]!r}, bound {bound[bad][0]!r}")


class Scene:
    """A cache with prefixes and requests on scattered pages: every row that no key owns is NaN or infinite."""

    def __init__(self, requests, prefixes, heads, kv_heads, D, P, dtype, seed, layers=1, pad_rows=(), order=None, std_q=1.0, device="cuda"):
        """requests: (prefix or -1, own keys) each; one token per request, at its last position."""
        import mlora
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.P, self.D, self.dtype, self.heads, self.kv_heads = P, D, dtype, heads, kv_heads
        counts = [-(-n // P) for n in prefixes] + [-(-n // P) for _, n in requests]
        n_pages = sum(counts) + 5
        ids = rng.permutation(n_pages)
        lists, at = [], 0
        for c in counts:
            lists.append([int(i) for i in ids[at:at + c]])
            at += c
        self.prefix_lists, self.req_lists = lists[:len(prefixes)], lists[len(prefixes):]
        self.prefixes, self.requests = list(prefixes), list(requests)
        self.cache = mlora.KVCache(layers, n_pages, kv_heads, D, page_tokens=P, dtype=dtype, device=device)
        self.k = torch.full(tuple(self.cache.k.shape), float("nan"), dtype=dtype)
        self.v = torch.full(tuple(self.cache.v.shape), float("nan"), dtype=dtype)
        self.v[:, :, :, 1::2] = float("inf")
        for pages, n in zip(lists, list(prefixes) + [n for _, n in requests]):
            for i in range(0, n, P):
                m = min(P, n - i)
                for t in (self.k, self.v):
                    t[:, pages[i // P], :, :m] = torch.randn((layers, kv_heads, m, D), generator=g).to(dtype)
        self.cache.k.copy_(self.k)
        self.cache.v.copy_(self.v)
        T = len(requests)
        order = list(range(T)) if order is None else order
        req, pos = [], []
        for r in order:
            f, n = requests[r]
            req.append(r)
            pos.append((prefixes[f] if f >= 0 else 0) + n - 1)
        for row in sorted(pad_rows):
            req.insert(row, -1)
            pos.insert(row, 7)
        self.req, self.pos = req, pos
        i32 = dict(dtype=torch.int32, device=device)
        table = lambda ls: torch.tensor([l + [-1] * (max(1, max(map(len, ls))) - len(l)) for l in ls], **i32)   # noqa: E731
        self.batch = mlora.KVBatch(torch.tensor(req, **i32), torch.tensor(pos, **i32), table(self.req_lists),
                                   torch.tensor([f for f, _ in requests], **i32) if prefixes else None,
                                   table(self.prefix_lists) if prefixes else None,
                                   torch.tensor(prefixes, **i32) if prefixes else None)
        self.q = (torch.randn((len(req), heads, D), generator=g) * std_q).to(dtype)
        self.dev_q = self.q.to(device)

    def rows(self, which, layer, pages, n, head):
        t = (self.k if which == "k" else self.v)[layer]
        n = min(n, len(pages) * self.P)
        keep = [i for i in range(n) if 0 <= pages[i // self.P] < t.shape[0]]
        return np.stack([f64(t[pages[i // self.P], head, i % self.P]) for i in keep]) if keep else np.zeros((0, self.D))

    def exact(self, t, head, layer=0, scale=None):
        """Row of token t (with a request) and query head."""
        scale = self.D ** -0.5 if scale is None else scale
        r, pos = self.req[t], self.pos[t]
        kv = head // (self.heads // self.kv_heads)
        f = self.requests[r][0]
        base = self.prefixes[f] if f >= 0 else 0
        parts = {"k": [], "v": []}
        for w in "kv":
            if f >= 0:
                parts[w].append(self.rows(w, layer, self.prefix_lists[f], min(base, pos + 1), kv))
            parts[w].append(self.rows(w, layer, self.req_lists[r], max(0, pos + 1 - base), kv))
        return attention_exact(f64(self.q[t, head]), np.concatenate(parts["k"]), np.concatenate(parts["v"]), scale, self.dtype)

    def compare(self, got, layer=0, scale=None, tokens=None, heads=None, what=""):
        for t in (range(len(self.req)) if tokens is None else tokens):
            if self.req[t] < 0:
                continue
            for h in (range(self.heads) if heads is None else heads):
                want, bound = self.exact(t, h, layer, scale)
                check(got[t, h], want, bound, f"{what} token {t} (request {self.req[t]}, position {self.pos[t]}) head {h}")
