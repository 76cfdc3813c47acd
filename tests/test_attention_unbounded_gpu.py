"""Infinities and NaNs among the keys' values where rows do see them: every row's output is the formula's (the infinity, or
NaN), wherever the key lies in the tiles, and everything else keeps its bits."""
import math

import numpy as np
import pytest

import splash_q4 as sq
from attention_oracle import Cache, bf16, run_attention, torch

pytestmark = pytest.mark.gpu


def queries(rng, c, heads, dim):
    return bf16(rng.standard_normal((c.rows, heads, dim)))


def check_bits(got, clean, at, what):
    """got is clean's bits but where `at` (columns of rows and heads) says."""
    same = np.array_equal(got[~at], clean[~at])
    assert same, f"{what}: {np.sum(got[~at] != clean[~at])} other values changed"


# (heads, key heads, head_dim, (rows, keys) of each sequence, the plan's tile)
TILES = [
    (4, 2, 64, [(1, 300)], 16), (4, 1, 128, [(1, 700), (1, 90)], 16), (8, 2, 128, [(1, 20001)], 16),
    (6, 2, 80, [(3, 1500)], 16), (16, 2, 256, [(2, 3000), (1, 70)], 16), (2, 2, 16, [(1, 200)], 16),
    (8, 2, 64, [(8, 700), (3, 64)], 32), (16, 2, 128, [(4, 9000)], 32), (5, 1, 96, [(6, 400)], 32),
    (8, 2, 64, [(70, 333)], 128), (8, 2, 128, [(100, 900), (1, 500)], 128), (4, 1, 256, [(64, 3000)], 128),
]


@pytest.mark.parametrize("heads,kv_heads,dim,sizes,tile", TILES)
def test_seen_infinities(heads, kv_heads, dim, sizes, tile):
    """Infinite values of early keys, which every row of their tile sees, and of the last ones."""
    rng = np.random.default_rng(dim + heads)
    clean, bad = (Cache(np.random.default_rng(7), sizes, kv_heads, dim, 16, "bf16") for _ in range(2))
    plan = sq.attention_plan(sq.AttentionShape(heads, clean.shape, 1, 0, 1 / math.sqrt(dim)), len(sizes), clean.rows,
                             max(r for r, _ in sizes))
    assert plan.tile_rows == tile
    n, keys = sizes[0]
    first = keys - n                                  # the first row's position
    want = {}                                         # column of the last key head -> what every row has there
    for column, value, key in ((0, np.inf, 3), (5, -np.inf, first // 2), (dim - 1, np.inf, first - 1), (9, np.inf, first)):
        bad.v[0][-1, key, column] = value
        want[column] = value
    bad.v[0][-1, 4, 12], bad.v[0][-1, first // 3, 12], want[12] = np.inf, -np.inf, np.nan
    q = queries(rng, clean, heads, dim)
    a, b = (run_attention(c.fill(), q, 1 / math.sqrt(dim), plan=plan) for c in (clean, bad))
    group = heads // kv_heads
    changed = np.zeros(b.shape, bool)
    for column, value in want.items():
        changed[:n, heads - group:, column] = True
        got = b[:n, heads - group:, column]
        assert np.array_equal(got, np.full_like(got, value), equal_nan=True), (column, value, got)
    check_bits(b, a, changed, tile)


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("heads,kv_heads,dim,sizes,tile", TILES)
def test_nan_codes(heads, kv_heads, dim, sizes, tile, window):
    """E4M3's NaN codes under finite scales (no write makes them, but pages may be filled by others, or not yet): the rows
    that see such a value have NaN in its column, the rows before it or past whose window it lies keep their bits."""
    t = torch()
    rng = np.random.default_rng(dim + heads)
    clean, bad = (Cache(np.random.default_rng(7), sizes, kv_heads, dim, 16, "e4m3").fill() for _ in range(2))
    plan = sq.attention_plan(sq.AttentionShape(heads, clean.shape, 1, window, 0.1), len(sizes), clean.rows,
                             max(r for r, _ in sizes))
    assert plan.tile_rows == tile
    n, keys = sizes[0]
    first, group = keys - n, heads // kv_heads
    position = np.arange(first, keys)
    nan = np.zeros((clean.rows, heads, dim), bool)

    def put(tensor, head, key, column, code):
        page, slot = bad.slot(0, key)
        tensor.view(t.uint8)[int(page), head, slot, column] = code
        sees = (key <= position) & (key > position - (window or keys))
        columns = [column] if tensor is bad.values else range(dim)
        for r in np.flatnonzero(sees):
            nan[r, head * group:(head + 1) * group, columns] = True

    put(bad.values, kv_heads - 1, keys - 2, 3, 0x7F)
    put(bad.values, kv_heads - 1, keys - 1, dim - 1, 0xFF)
    put(bad.values, kv_heads - 1, first, 8, 0x7F)
    put(bad.values, kv_heads - 1, 3, 7, 0xFF)
    put(bad.values, kv_heads - 1, max(0, first - 36), 5, 0xFF)     # with the window: the first four rows see it
    if kv_heads > 1:
        put(bad.keys, 0, keys - 1, 2, 0x7F)
    q = queries(rng, clean, heads, dim)
    a, b = (run_attention(c, q, 0.1, window=window, plan=plan) for c in (clean, bad))
    assert np.isnan(b[nan]).all(), f"{np.sum(~np.isnan(b[nan]))} of {nan.sum()} that see a NaN have none"
    check_bits(b, a, nan, tile)
