"""Paged batches, and the cache append, paged attention and sampling in 64
bits with numpy: the definitions that the GPU tests compare with."""
from __future__ import annotations

import math

import numpy as np

F32, F16, BF16 = 0, 1, 30
# half a step of a type, relative to the value
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
# and where values get too small for that, of the smallest ones
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}


def encode(x, kind):
    """float array -> the type's bits (nearest, ties to even)."""
    x = np.asarray(x, np.float32)
    if kind == F32:
        return x.view(np.uint32)
    if kind == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32)
    rounded = ((b.astype(np.uint64) + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), rounded)


def decode(bits, kind):
    """the type's bits -> float64."""
    if kind == F32:
        return bits.view(np.float32).astype(np.float64)
    if kind == F16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Paged:
    """A cache and a batch of sequences with `new` tokens each, `contexts` long:
    host arrays, and the same on the device after upload()."""

    def __init__(self, new, contexts, *, kv_heads=2, dim=64, page=16, kind=F16, head_major=False, seed=1, gaps=(0, 0),
                 spare=2, extra_entries=0):
        rng = np.random.default_rng(seed)
        self.rng, self.new, self.contexts = rng, list(new), list(contexts)
        self.kv_heads, self.dim, self.page, self.kind, self.head_major = kv_heads, dim, page, kind, head_major
        self.tokens = gaps[0] + sum(new) + gaps[1]  # rows that no sequence owns at both ends
        self.start = (gaps[0] + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)
        held = [-(-c // page) for c in contexts]
        self.pages = sum(held) + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(new), max(1, max(held, default=1)) + extra_entries), -7, np.int32)
        at = 0
        for s, n in enumerate(held):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (self.pages, kv_heads, page, dim) if head_major else (self.pages, page, kv_heads, dim)
        self.k, self.v = (encode(rng.standard_normal(shape), kind) for _ in range(2))

    def strides(self):
        H, P, D = self.kv_heads, self.page, self.dim
        return (H * P * D, D, P * D) if self.head_major else (H * P * D, H * D, D)

    def seen(self, pool):
        """The pool as [page, slot, head, dim]."""
        return pool.transpose(0, 2, 1, 3) if self.head_major else pool

    def rows(self, s, pool):
        """A sequence's cached rows [context, heads, dim] (bits)."""
        c = self.contexts[s]
        pages = self.table[s, :-(-c // self.page)] if c else self.table[s, :0]
        return self.seen(pool)[pages].reshape(-1, self.kv_heads, self.dim)[:c]

    def upload(self, qk):
        b = qk.DeviceBuffer.from_array
        self.dev = {"k": b(self.k), "v": b(self.v), "start": b(self.start),
                    "context": b(np.asarray(self.contexts, np.int32)), "table": b(self.table),
                    "fault": b(np.zeros(1, np.uint32))}
        d = self.dev
        ps, ts, hs = self.strides()
        self.cache = qk.KVCache(k=d["k"].ptr, v=d["v"].ptr, type=self.kind, pages=self.pages, page_size=self.page,
                                kv_heads=self.kv_heads, head_dim=self.dim, page_stride=ps, token_stride=ts,
                                head_stride=hs, fault=d["fault"].ptr)
        self.batch = qk.KVBatch(sequences=len(self.new), tokens=self.tokens, token_start=d["start"].ptr,
                                context=d["context"].ptr, page_table=d["table"].ptr, table_stride=self.table.shape[1])
        return self

    def fault(self):
        return int(self.dev["fault"].download(np.uint32)[0])


def rotate(x, positions, weight, eps, base, dims, interleaved):
    """x [tokens, heads, dim] in 64 bits: the head norm, then the rotation."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    if dims == 0:
        return x.copy()
    j = np.arange(dims // 2)
    angle = np.asarray(positions, np.float64)[:, None] * float(base) ** (-2.0 * j / dims)
    c, n = np.cos(angle)[:, None], np.sin(angle)[:, None]
    lo, hi = (slice(0, dims, 2), slice(1, dims, 2)) if interleaved else (slice(0, dims // 2), slice(dims // 2, dims))
    out = x.copy()
    out[..., lo] = x[..., lo] * c - x[..., hi] * n
    out[..., hi] = x[..., hi] * c + x[..., lo] * n
    return out


def pair_size(x, dims, interleaved):
    """The length of the pair that each value rotates in (itself where it does not)."""
    out = np.abs(x)
    if dims:
        lo, hi = (slice(0, dims, 2), slice(1, dims, 2)) if interleaved else (slice(0, dims // 2), slice(dims // 2, dims))
        size = np.hypot(x[..., lo], x[..., hi])
        out[..., lo], out[..., hi] = size, size
    return out


def attention(q, K, V, first, scale, window):
    """One sequence: q [n, heads, dim] at positions first .. against K, V
    [context, kv heads, dim] (float64). Returns out, lse, and what a tolerance
    is made of: sum p|v| per value and the largest sum |q k| of a row. Masked
    keys are left out of every sum, whatever they hold."""
    n, H, D = q.shape
    G = H // K.shape[1]
    out, lse = np.zeros((n, H, D)), np.full((n, H), -np.inf)
    weight, reach = np.zeros((n, H, D)), np.zeros((n, H))
    for i in range(n):
        t = first + i
        lo = max(0, t - window + 1) if window else 0
        hi = min(t + 1, K.shape[0])
        if hi <= lo:
            continue
        for h in range(H):
            k, v = K[lo:hi, h // G], V[lo:hi, h // G]
            s = scale * (k @ q[i, h])
            m = s.max()
            p = np.exp(s - m)
            out[i, h] = p @ v / p.sum()
            lse[i, h] = m + math.log(p.sum())
            weight[i, h] = p @ np.abs(v) / p.sum()
            reach[i, h] = abs(scale) * (np.abs(k) @ np.abs(q[i, h])).max()
    return out, lse, weight, reach


def sample(z, heat, k, p, min_p, u):
    """One row: (token, probability, kept indices, weights)."""
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    if z.max() == -np.inf:
        return 0xFFFFFFFF, 0.0
    if not heat > 0:
        return int(z.argmax()), 1.0
    order = np.argsort(-z, kind="stable")
    order = order[z[order] > -np.inf]
    if k > 0:
        order = order[:k]
    top = z[order[0]]
    w = np.where(z[order] == top, 1.0, np.exp((np.where(z[order] == top, 0.0, z[order]) - (0 if np.isinf(top) else top))
                                              / float(heat)))
    if np.isinf(top):
        w = (z[order] == top).astype(np.float64)
    if p < 1:
        before = np.cumsum(w) - w
        n = max(1, int((before < float(p) * w.sum()).sum()))
        order, w = order[:n], w[:n]
    stay = w >= min_p
    stay[0] = True
    order, w = order[stay], w[stay]
    by = np.argsort(order)
    order, w = order[by], w[by]
    run = np.cumsum(w)
    at = min(int(np.searchsorted(run, float(u) * run[-1], side="right")), len(w) - 1)
    while w[at] == 0:
        at -= 1
    return int(order[at]), float(w[at] / run[-1])
