"""The 4-bit cache's codes and scales in 64 bits (numpy), and batches over such a cache for the GPU tests."""
from __future__ import annotations

import numpy as np

import splash_q4 as sq
from attention_oracle import Cache, torch

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def scale_bytes(dim):
    return 2 if dim <= 64 else 4 if dim <= 128 else 8


def quantised4(x):
    """(codes [..., dim], scale bytes [..., 2, 4 or 8]) of head rows [..., dim] of bf16 values: every step is exact in 64
    bits."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = np.abs(g).max(-1)
    bad = ~np.isfinite(top)
    top = np.where(bad, 1.0, top)
    mantissa, e = np.frexp(top)                               # top = mantissa 2^e, mantissa in [1/2, 1)
    e = np.clip(np.where(top > 0, e - 3 + (mantissa > 0.875), -1000), -125, 125)   # least with top <= 7 2^e
    with np.errstate(invalid="ignore"):
        q = np.where(bad[..., None], 0.0, np.ldexp(g, -e[..., None]))
    size = np.abs(q)
    hi = np.clip(np.searchsorted(E2M1, size), 1, 7)
    below, above = size - E2M1[hi - 1], E2M1[hi] - size
    code = np.where(below < above, hi - 1, np.where(above < below, hi, np.where(hi % 2 == 0, hi, hi - 1)))
    code = (code + 8 * (np.signbit(q) & ~bad[..., None])).astype(np.uint8)
    scales = np.full((*x.shape[:-1], scale_bytes(x.shape[-1])), 2, np.uint8)
    scales[..., :x.shape[-1] // 32] = np.where(bad, 255, e + 127)
    return code.reshape(x.shape), scales


def packed(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def values4(codes, scales):
    """What codes [..., dim] and scale bytes stand for, rounded to bf16 where that matters (past its range)."""
    g = codes.reshape(*codes.shape[:-1], codes.shape[-1] // 32, 32)
    by = scales[..., :g.shape[-2], None].astype(np.int64)
    v = np.ldexp(np.where(g & 8, -1.0, 1.0) * E2M1[g & 7], by - 127)
    v = np.where(by == 255, np.nan, np.where(np.abs(v) >= 2.0 ** 128, np.copysign(np.inf, v), v))
    return v.reshape(codes.shape)


class Cache4(Cache):
    """A paged cache in 4 bits and a batch over it; every page slot that no key of the batch lives in holds NaN."""

    def __init__(self, rng, sizes, kv_heads, dim, page, **kw):
        super().__init__(rng, sizes, kv_heads, dim, page, "bf16", **kw)
        t = torch()
        self.fmt = "e2m1"
        self.shape = sq.KvShape(kv_heads, dim, page, sq.KV_E2M1)
        rows = (self.pages, kv_heads, page)
        make = lambda width: t.full((*rows, width), 255, dtype=t.uint8, device="cuda")  # noqa: E731
        self.keys, self.values = make(dim // 2), make(dim // 2)
        self.key_scales, self.value_scales = make(scale_bytes(dim)), make(scale_bytes(dim))

    def struct(self):
        return sq.kv_cache(self.shape, self.pages, self.keys, self.values, self.key_scales, self.value_scales)

    def fill(self):
        t = torch()
        for name, parts in (("key", self.k), ("value", self.v)):
            codes, scales = (getattr(self, name + n).cpu().numpy() for n in ("s", "_scales"))
            for s, part in enumerate(parts):
                at = np.arange(part.shape[1])
                if len(at):
                    c, f = quantised4(part)
                    pages, slots = self.table[s, at // self.page], at % self.page
                    codes[pages, :, slots] = np.moveaxis(packed(c), 1, 0)
                    scales[pages, :, slots] = np.moveaxis(f, 1, 0)
            setattr(self, name + "s", t.from_numpy(codes).cuda())
            setattr(self, name + "_scales", t.from_numpy(scales).cuda())
        return self

    def stored(self, s):
        return [values4(*quantised4(part)) for part in (self.k[s], self.v[s])]
