"""Attention with capped and biased scores, first keys and prefixes, in 64 bits (numpy), and the library's call."""
from __future__ import annotations

import numpy as np

import splash_q4 as sq
from attention_oracle import HALF_STEP, from_bf16, to_bf16, torch


def scored_f64(q, cache, scale, causal=True, window=0, cap=0.0, slopes=None, begins=None, prefixes=None):
    """q [rows, heads, dim] -> (outputs, their bounds) [live rows, heads, dim].

    The bound is the plain one's (attention_oracle: the weights and the output rounded to bf16, scores as sums of dim products
    in fp32, fp32 sums of keys / 32 + 64 in a chain), with a score's error key by key: the cap's own, 2^-21 of a cap up to 128
    or 2^-20 of the score; of a bias three roundings (the slope times log2 e, the product, the sum), 3 2^-24 of it and of the
    score; and 2^-22 of both the score and the row's largest (their difference and its exponential)."""
    rows, heads, dim = cache.live_rows, q.shape[1], q.shape[2]
    group = heads // cache.kv_heads
    out, bound = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim))
    for s, (n, keys) in enumerate(cache.sizes):
        if not n or not keys:
            continue
        k, v = cache.stored(s)
        at, j = np.arange(keys - n, keys)[:, None], np.arange(keys)[None]
        sees = np.ones((n, keys), bool)
        if causal:
            sees = j <= at
            if prefixes is not None:
                sees = sees | ((j < prefixes[s]) & (at >= 0))
        if begins is not None:
            sees = sees & (j >= begins[s])
        if window:
            sees = sees & (j > at - window)
        for h in range(heads):
            x = q[cache.starts[s]:cache.starts[s + 1], h]
            kh, vh = k[h // group], np.where(np.isfinite(v[h // group]), v[h // group], 0.0)
            with np.errstate(invalid="ignore"):
                t = np.where(sees, (x @ kh.T) * scale, 0.0)
            error = (dim + 4) * 2.0 ** -24 * np.where(sees, np.abs(x) @ np.abs(kh).T * abs(scale), 0.0)
            if cap:
                t = cap * np.tanh(t / cap)
                error = error + (cap * 2.0 ** -21 if cap <= 128 else 2.0 ** -20 * np.abs(t))
            if slopes is not None:
                bias = slopes[h] * np.abs(at - j)
                t = t - bias
                error = error + 3 * 2.0 ** -24 * (np.abs(bias) + np.abs(t))
            t = np.where(sees, t, -np.inf)
            top = t.max(-1, keepdims=True)
            top = np.where(np.isfinite(top), top, 0.0)
            p = np.where(sees, np.exp(t - top), 0.0)
            total = p.sum(-1, keepdims=True)
            p /= np.where(total > 0, total, 1.0)
            with np.errstate(invalid="ignore"):
                error = np.where(sees, np.expm1(error + 2.0 ** -22 * (np.abs(t) + np.abs(top))), 0.0)
            o, size = p @ vh, p @ np.abs(vh)
            # Below fp32's normal range all of a number may go: of a weight (an exponential of 2^-126 or less is zero; the row's
            # largest is 1 or more), of what it lost to its first bf16, of its products' sum on its way from one running maximum
            # to the next or out of a part (three more factors), each at most 2^-126 a value of |v|.
            lost = 5 * 2.0 ** -126 * np.where(sees, 1.0, 0.0) @ np.abs(vh)
            off = (p * error) @ np.abs(vh) + np.abs(o) * (p * error).sum(-1, keepdims=True) + lost
            at_rows = slice(cache.starts[s], cache.starts[s + 1])
            out[at_rows, h] = o
            bound[at_rows, h] = HALF_STEP * np.abs(o) + (size * (HALF_STEP + (keys / 32 + 64) * 2.0 ** -24) + off) * (1 + HALF_STEP)
    return out, bound


def device_words(values):
    return torch().from_numpy(np.asarray(values, np.uint32).view(np.int32)).cuda()


def scores_of(cap=0.0, slopes=None, begins=None, prefixes=None):
    """(the call's struct, the tensors that it points to)."""
    t = torch()
    keep = [t.tensor(slopes, dtype=t.float32, device="cuda") if slopes is not None else None,
            device_words(begins) if begins is not None else None, device_words(prefixes) if prefixes is not None else None]
    return sq.attention_scores(cap, *keep), keep


def run_scored(cache, q, scale, causal=True, window=0, chunk=None, **what):
    """The library's outputs [rows, heads, dim] (rows behind the last sequence included)."""
    t = torch()
    rows, heads, _ = q.shape
    shape = sq.AttentionShape(heads, cache.shape, int(causal), window, scale)
    plan = sq.attention_plan(shape, len(cache.sizes), rows, min(chunk or max([r for r, _ in cache.sizes] + [1]), rows))
    scores, keep = scores_of(**what)
    out = t.full((rows, heads * q.shape[2]), 123.0, dtype=t.bfloat16, device="cuda")
    sq.attention_add(plan, cache.struct(), cache.batch(), to_bf16(q.reshape(rows, -1)), out, sq.AttentionScratch(plan),
                     scores=scores)
    t.cuda.synchronize()
    return from_bf16(out).reshape(q.shape)
