"""Caches of Q4_1 blocks on the host: the blocks' format with numpy, and a paged
batch over such a cache (its k and v are the F16 bits that the blocks stand for,
so that every definition of an F16 cache holds for it)."""
from __future__ import annotations

import numpy as np

import serving_ref as ref
from serving_ref import F16, Paged

Q4_1 = 3


def blocks_of(x):
    """fp32 [.., D] -> bytes [.., D / 32 * 20], every step in fp32 as the format's definition has it."""
    x = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        low, high = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
        m = low.astype(np.float16)
        span = np.maximum(high - m.astype(np.float32), np.float32(0)) / np.float32(15)
        d = span.astype(np.float16)
        d = np.where(d.astype(np.float32) > span, (d.view(np.uint16) - 1).astype(np.uint16).view(np.float16), d)
        step = d.astype(np.float32)
        inverse = np.where(step == 0, np.float32(0), np.float32(1) / step)
        code = np.clip(np.rint((x - m.astype(np.float32)) * inverse), 0, 15)
        broken = ~(np.isfinite(m) & np.isfinite(high.astype(np.float16)) & ~np.isnan(x).any(-1, keepdims=True))
    code = np.where(broken, 0, code).astype(np.uint8)
    nan = np.uint16(0x7E00)
    d, m = (np.where(broken, nan, y.view(np.uint16)).astype(np.uint16) for y in (d, m))
    out = np.concatenate([d.view(np.uint8), m.view(np.uint8), code[..., :16] | code[..., 16:] << 4], -1)
    return np.ascontiguousarray(out.reshape(*x.shape[:-2], -1))


def parts(blocks):
    """(d, m, codes [.., 32]) of blocks [.., n], the first two float64 with a last axis of 1."""
    b = np.ascontiguousarray(blocks).reshape(*blocks.shape[:-1], -1, 20)
    dm = np.ascontiguousarray(b[..., :4]).view(np.float16).astype(np.float64)
    return dm[..., :1], dm[..., 1:], np.concatenate([b[..., 4:] & 15, b[..., 4:] >> 4], -1)


def values(blocks):
    """F16 bits of what blocks stand for: d * code + m (exact in 64 bits), rounded once."""
    d, m, code = parts(blocks)
    with np.errstate(over="ignore", invalid="ignore"):
        v = (d * code + m).astype(np.float16).view(np.uint16)
    return v.reshape(*blocks.shape[:-1], -1)


class Paged4(Paged):
    """A Q4_1 cache of random values; k4 and v4 are its bytes. After a change of those, settle()."""

    def __init__(self, new, contexts, *, kind=F16, **more):
        assert kind == F16
        super().__init__(new, contexts, kind=F16, **more)
        self.k4, self.v4 = (blocks_of(ref.decode(x, F16).astype(np.float32)) for x in (self.k, self.v))
        self.settle()

    def settle(self):
        self.k, self.v = values(self.k4), values(self.v4)
        return self

    def spoil(self, pool4, where):
        """NaN in all values of the rows `where` of seen(pool4)."""
        rows = self.seen(pool4)
        block = np.zeros(20, np.uint8)
        block[:4] = np.array([0x7E00, 0x7E00], np.uint16).view(np.uint8)
        rows[where] = np.tile(block, self.dim // 32)

    def upload(self, qk):
        super().upload(qk)
        for n, x in (("k", self.k4), ("v", self.v4)):
            self.dev[n] = qk.DeviceBuffer.from_array(x)
        self.cache.k, self.cache.v, self.cache.type = self.dev["k"].ptr, self.dev["v"].ptr, Q4_1
        return self

    def downloaded(self, name):
        """Bytes of a pool as they are on the device, shaped as k4."""
        return self.dev[name].download(np.uint8).reshape(self.k4.shape)
