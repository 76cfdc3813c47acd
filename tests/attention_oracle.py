"""The definitions of rotary positions, the paged cache and attention in 64 bits (numpy), and the batches their GPU tests
run on."""
from __future__ import annotations

import math

import numpy as np

import splash_q4 as sq
from splash_q4 import synthetic

HALF_STEP = 2.0 ** -8       # of bf16: torch.finfo(torch.bfloat16).eps / 2
FORMATS = {"bf16": sq.KV_BF16, "int8": sq.KV_INT8, "e4m3": sq.KV_E4M3}
TOP = {"int8": 127.0, "e4m3": 448.0}


def torch():
    import torch as t
    return t


def bf16(x):
    """float array -> the bf16 values nearest to it, as float64."""
    return synthetic.bf16_to_f32(synthetic.bf16_bits(np.asarray(x, np.float32))).astype(np.float64)


def to_bf16(x):
    """float64 values that are bf16 -> a device tensor of them."""
    return torch().from_numpy(np.ascontiguousarray(x, np.float32)).to(torch().bfloat16).cuda()


def from_bf16(tensor):
    return tensor.float().cpu().numpy().astype(np.float64)


# ---------------------------------------------------------------- rope

def rope_f64(x, positions, frequencies, magnitude, interleaved):
    """x [rows, heads, dim] rotated; positions [rows]. Also sum |x| of each value's pair (the error's scale)."""
    n = len(frequencies)
    turns = np.multiply.outer(np.asarray(positions, np.float64), np.asarray(frequencies))[:, None]
    c, s = np.cos(turns) * magnitude, np.sin(turns) * magnitude
    y, scale = x.copy(), np.abs(x)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    scale[..., a] = scale[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * abs(magnitude)
    return y, scale


def rope_bound(y, scale):
    """One rounding to bf16, and fp32 before it: a cosine or sine off by 2^-22 (the fraction of a turn rounded to fp32 is
    off by 2^-25 turns, 2^-22.3 radians; the function 2 units of 2^-24), three roundings of products and their sum."""
    return HALF_STEP * np.abs(y) + scale * (2 ** -22 + 5 * 2 ** -24) * (1 + HALF_STEP)


# ---------------------------------------------------------------- cache

E4M3 = np.array([m * 2.0 ** -9 for m in range(8)] +
                [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)])


def nearest_e4m3(q):
    """The code's value nearest to q; of two as near, the even code."""
    magnitude = np.abs(q)
    hi = np.clip(np.searchsorted(E4M3, magnitude), 1, len(E4M3) - 1)
    below, above = magnitude - E4M3[hi - 1], E4M3[hi] - magnitude
    pick = np.where(below < above, hi - 1, np.where(above < below, hi, np.where(hi % 2 == 0, hi, hi - 1)))
    return np.copysign(E4M3[pick], q)


def quantised(x, fmt):
    """(code values, fp32 scales) of head rows [..., dim] of bf16 values. x top is exact in 64 bits and ties are exactly
    representable, so the quotient's rounding does not move a code."""
    if fmt == "bf16":
        return x, np.ones(x.shape[:-1], np.float32)
    m = np.abs(x).max(-1)
    with np.errstate(invalid="ignore", divide="ignore"):
        q = x * TOP[fmt] / np.where(m > 0, m, 1)[..., None]
    bad = ~np.isfinite(m)
    q = np.where(bad[..., None], 0.0, q)
    codes = np.rint(q) if fmt == "int8" else nearest_e4m3(q)
    with np.errstate(invalid="ignore"):
        scale = np.where(bad, np.float32(np.nan), m.astype(np.float32) / np.float32(TOP[fmt]))
    return codes, scale.astype(np.float32)


class Cache:
    """A paged cache and a batch over it. sizes: (new rows, keys with them) of each sequence. Every page slot that no key
    of the batch lives in holds NaN (8-bit: the e4m3 NaN code and NaN scales)."""

    def __init__(self, rng, sizes, kv_heads, dim, page, fmt, extra_rows=0, spare_pages=3, key_scale=1.0):
        t = torch()
        self.sizes, self.kv_heads, self.dim, self.page, self.fmt = sizes, kv_heads, dim, page, fmt
        most = max(1, max(-(-k // page) for _, k in sizes) + 1)
        used = sum(-(-k // page) for _, k in sizes)
        self.pages = used + spare_pages
        order, at = rng.permutation(self.pages), 0
        self.table = np.full((len(sizes), most), 0xFFFFFFFF, np.uint32)
        for s, (_, k) in enumerate(sizes):
            n = -(-k // page)
            self.table[s, :n] = order[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum([r for r, _ in sizes])]).astype(np.uint32)
        self.lengths = np.array([k for _, k in sizes], np.uint32)
        self.live_rows, self.rows = int(self.starts[-1]), int(self.starts[-1]) + extra_rows
        # The sequences' keys and values as bf16, before they are stored: [heads, keys, dim] each.
        channels = 1 + 3 * (rng.random((kv_heads, 1, dim)) > 0.9)
        self.k = [bf16(rng.standard_normal((kv_heads, n, dim)) * channels * key_scale) for _, n in sizes]
        self.v = [bf16(rng.standard_normal((kv_heads, n, dim))) for _, n in sizes]
        self.shape = sq.KvShape(kv_heads, dim, page, FORMATS[fmt])
        pool = (self.pages, kv_heads, page, dim)
        kind = {"bf16": t.bfloat16, "int8": t.int8, "e4m3": t.float8_e4m3fn}[fmt]
        empty = t.full(pool, math.nan if fmt != "int8" else 77.0).to(kind).cuda()
        self.keys, self.values = empty.clone(), empty.clone()
        scales = t.full(pool[:3], math.nan, dtype=t.float32, device="cuda")
        self.key_scales, self.value_scales = scales.clone(), scales.clone()
        self.starts_d, self.lengths_d, self.table_d = (
            t.from_numpy(a.view(np.int32)).cuda() for a in (self.starts, self.lengths, self.table))

    def struct(self):
        return sq.kv_cache(self.shape, self.pages, self.keys, self.values,
                           *((self.key_scales, self.value_scales) if self.fmt != "bf16" else ()))

    def batch(self):
        return sq.kv_batch(self.starts_d, self.lengths_d, self.table_d, self.rows)

    def slot(self, s, position):
        return self.table[s, position // self.page], position % self.page

    def fill(self):
        """Stores every sequence's keys and values in its pages, from the host."""
        t = torch()
        stored = {}
        for name, parts in (("key", self.k), ("value", self.v)):
            codes = getattr(self, name + "s").float().cpu().numpy()
            scales = getattr(self, name + "_scales").cpu().numpy()
            for s, part in enumerate(parts):
                c, f = quantised(part, self.fmt)
                at = np.arange(part.shape[1])
                if len(at):
                    pages, slots = self.table[s, at // self.page], at % self.page
                    codes[pages, :, slots] = np.moveaxis(c, 1, 0)
                    scales[pages, :, slots] = np.moveaxis(f, 1, 0)
            kind = getattr(self, name + "s").dtype
            setattr(self, name + "s", t.from_numpy(codes).to(kind).cuda())
            setattr(self, name + "_scales", t.from_numpy(scales).cuda())
        return self

    def stored(self, s):
        """(keys, values) of sequence s as the cache's format holds them, in 64 bits."""
        out = []
        for part in (self.k[s], self.v[s]):
            c, f = quantised(part, self.fmt)
            out.append(c * (f.astype(np.float64)[..., None] if self.fmt != "bf16" else 1.0))
        return out

    def new_rows(self, part):
        """The batch's rows [rows, heads * dim] of `part` (self.k or self.v): each sequence's last rows."""
        out = np.zeros((self.rows, self.kv_heads, self.dim))
        for s, (n, keys) in enumerate(self.sizes):
            have = min(n, keys)
            if have:
                out[self.starts[s + 1] - have:self.starts[s + 1]] = np.moveaxis(part[s][:, keys - have:], 1, 0)
        return out.reshape(self.rows, -1)


# ---------------------------------------------------------------- attention

def attention_f64(q, cache, scale, causal=True, window=0, hidden=None):
    """q [rows, heads, dim] -> (outputs, their bounds) [live rows, heads, dim]. hidden(s, position) -> keys of sequence
    s that no row sees (holes).

    The bound: the weights are rounded to bf16 (half a step each, so HALF_STEP of sum p |v|) and the output once more.
    A score is a sum of dim products in fp32, off by at most (dim + 4) 2^-24 sum |q k| scale (the 8-bit formats' scale
    is one more rounding), and its exponential another 2^-22 of the score's size; a weight is off by e^that, in both
    directions within the sums, and the sums of fp32 weights and products by 2^-24 a key added one after the other in
    chains of at most keys / 32 + 64."""
    rows, heads, dim = cache.live_rows, q.shape[1], q.shape[2]
    group = heads // cache.kv_heads
    out, bound = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim))
    for s, (n, keys) in enumerate(cache.sizes):
        if not n:
            continue
        k, v = cache.stored(s)
        at = np.arange(keys - n, keys)[:, None]
        j = np.arange(keys)[None]
        sees = np.ones((n, keys), bool) if not causal else j <= at
        if window:
            sees = sees & (j > at - window)
        if hidden is not None:
            sees = sees & ~hidden(s, j)
        for h in range(heads):
            x = q[cache.starts[s]:cache.starts[s + 1], h]
            kh, vh = k[h // group], v[h // group]
            with np.errstate(invalid="ignore"):
                t = np.where(sees, (x @ kh.T) * scale, -np.inf)
            if not keys:
                continue
            top = t.max(-1, keepdims=True)
            p = np.where(sees, np.exp(t - np.where(np.isfinite(top), top, 0.0)), 0.0)
            total = p.sum(-1, keepdims=True)
            p /= np.where(total > 0, total, 1.0)
            o = p @ np.where(np.isfinite(vh), vh, 0.0)
            size = p @ np.abs(np.where(np.isfinite(vh), vh, 0.0))
            products = np.where(sees, np.abs(x) @ np.abs(kh).T * abs(scale), 0.0).max(-1, keepdims=True)
            score = (dim + 4) * 2 ** -24 * products + 2 ** -22 * np.where(sees, np.abs(t), 0.0).max(-1, keepdims=True)
            slack = 2 * np.expm1(score) + (keys / 32 + 64) * 2 ** -24
            out[cache.starts[s]:cache.starts[s + 1], h] = o
            bound[cache.starts[s]:cache.starts[s + 1], h] = HALF_STEP * np.abs(o) + size * (HALF_STEP + slack) * (1 + HALF_STEP)
    return out, bound


def run_attention(cache, q, scale, causal=True, window=0, chunk=None, scratch=None, plan=None, out=None):
    """The library's outputs [rows, heads, dim] (rows behind the last sequence included) for q [rows, heads, dim]."""
    t = torch()
    rows, heads, dim = q.shape
    shape = sq.AttentionShape(heads, cache.shape, int(causal), window, scale)
    chunk = chunk or max([r for r, _ in cache.sizes] + [1])
    plan = plan or sq.attention_plan(shape, len(cache.sizes), rows, min(chunk, rows))
    scratch = scratch or sq.AttentionScratch(plan)
    x = to_bf16(q.reshape(rows, -1))
    out = out if out is not None else t.full((rows, heads * dim), 123.0, dtype=t.bfloat16, device="cuda")
    sq.attention_add(plan, cache.struct(), cache.batch(), x, out, scratch)
    t.cuda.synchronize()
    return from_bf16(out).reshape(rows, heads, dim)


def check_attention(got, want, bound, what=""):
    err = np.abs(got - want)
    bad = ~(err <= bound)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} outside, worst {np.nanmax(err / np.maximum(bound, 1e-300)):.2f} "
                           f"of the bound, first at {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]}")
