"""Rotary positions, the paged cache and attention through the C ABI against their definitions in 64 bits: head sizes,
groups, formats, page sizes, ragged batches with empty sequences, windows, masks that leave a row nothing, NaN and
infinity where nobody looks, holes, graphs, streams, and the whole chain between the projections."""
import math

import numpy as np
import pytest

import splash_q4 as sq
from attention_oracle import (FORMATS, HALF_STEP, Cache, attention_f64, bf16, check_attention, from_bf16, quantised,
                              rope_bound, rope_f64, run_attention, to_bf16, torch)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- rope

def make_rope(rotary, interleaved=False, scaling=sq.ROPE_SCALING_NONE, base=1e4):
    layout = sq.ROPE_INTERLEAVED if interleaved else sq.ROPE_HALF
    c = sq.RopeConfig(rotary_dim=rotary, layout=layout, scaling=scaling, base=base, factor=8.0, original_positions=8192)
    return sq.RotaryPositions(c), *sq.rope_frequencies(c)


@pytest.mark.parametrize("rows,heads,dim,rotary,interleaved,scaling,far", [
    (1, 1, 16, 16, False, 0, 1), (1, 40, 128, 128, False, 0, 5000), (7, 3, 80, 40, False, 0, 300),
    (7, 3, 80, 40, True, 0, 300), (5, 9, 64, 2, False, 0, 100), (5, 9, 64, 6, True, 0, 100), (33, 5, 256, 256, False, 3, 4000000000),
    (33, 5, 256, 64, True, 3, 1000000), (130, 2, 96, 96, False, 2, 70000), (3, 17, 128, 100, False, 4, 100000),
    (3, 17, 128, 100, True, 1, 100000), (2, 6, 48, 48, False, 0, 1000),
])
def test_rope(rows, heads, dim, rotary, interleaved, scaling, far):
    t = torch()
    rng = np.random.default_rng(rows + dim + rotary)
    rope, f, magnitude = make_rope(rotary, interleaved, scaling)
    x = bf16(rng.standard_normal((rows, heads, dim)))
    positions = rng.integers(0, far, rows).astype(np.uint32)
    positions[0] = far - 1
    y, scale = rope_f64(x, positions, f, magnitude, interleaved)
    d, p = to_bf16(x.reshape(rows, -1)), t.from_numpy(positions.view(np.int32)).cuda()
    out = t.full_like(d, 9.0)
    sq.rope_add(rope, p, d, out, dim)
    got = from_bf16(out).reshape(x.shape)
    assert np.all(np.abs(got - y) <= rope_bound(y, scale)), np.abs(got - y).max()
    assert np.array_equal(got[..., rotary:], x[..., rotary:])
    # In place, and between columns of wider tensors: the same bits.
    sq.rope_add(rope, p, d, d, dim)
    wide_in, wide_out = (t.full((rows, heads * dim + 24), 5.0, dtype=t.bfloat16, device="cuda") for _ in range(2))
    wide_in[:, 16:16 + heads * dim] = to_bf16(x.reshape(rows, -1))
    sq.rope_add(rope, p, wide_in[:, 16:16 + heads * dim], wide_out[:, 8:8 + heads * dim], dim)
    t.cuda.synchronize()
    assert t.equal(d, out) and t.equal(wide_out[:, 8:8 + heads * dim], out)
    assert (wide_out[:, :8] == 5).all() and (wide_out[:, 8 + heads * dim:] == 5).all()


# ---------------------------------------------------------------- cache

SIZES = [(3, 3), (0, 40), (1, 100), (0, 0), (17, 50), (2, 33), (5, 3)]   # the last has rows before position 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kv_heads,dim,page", [(1, 16, 16), (3, 64, 32), (8, 128, 16), (2, 80, 64), (2, 256, 1024), (5, 144, 128)])
def test_write_and_read(fmt, kv_heads, dim, page):
    t = torch()
    rng = np.random.default_rng(dim + page)
    c = Cache(rng, SIZES, kv_heads, dim, page, fmt, extra_rows=2)
    for part, value in ((c.k, 1e-30), (c.v, 3e38)):     # magnitudes near both ends, and a row of zeros
        part[4][0, 40] = bf16(part[4][0, 40] * value / 8)
        part[4][0, 41] = 0.0
    k, v = c.new_rows(c.k), c.new_rows(c.v)
    width = kv_heads * dim
    fused = t.zeros((c.rows, 2 * width + 8), dtype=t.bfloat16, device="cuda")
    fused[:, :width], fused[:, width + 8:] = to_bf16(k), to_bf16(v)
    before = [x.clone() for x in (c.keys, c.values, c.key_scales, c.value_scales)]
    sq.kv_write(c.struct(), c.batch(), fused[:, :width], fused[:, width + 8:])
    outs = [t.full((c.rows, width), 7.0, dtype=t.bfloat16, device="cuda") for _ in range(2)]
    sq.kv_read(c.struct(), c.batch(), *outs)
    only = t.full((c.rows, width), 7.0, dtype=t.bfloat16, device="cuda")
    sq.kv_read(c.struct(), c.batch(), None, only)
    t.cuda.synchronize()
    assert t.equal(only, outs[1])
    written = np.zeros((c.pages, page), bool)
    for name, rows, out in (("key", k, outs[0]), ("value", v, outs[1])):
        codes, scales = quantised(rows.reshape(c.rows, kv_heads, dim), fmt)
        stored, stored_scales = getattr(c, name + "s").float().cpu().numpy(), getattr(c, name + "_scales").cpu().numpy()
        got = from_bf16(out).reshape(c.rows, kv_heads, dim)
        assert np.all(got[c.live_rows:] == 7.0), "rows behind the last sequence"
        for s, (n, keys) in enumerate(c.sizes):
            for i in range(n):
                r, position = int(c.starts[s]) + i, keys - n + i
                if position < 0:
                    assert np.all(got[r] == 0.0)
                    continue
                at, slot = c.slot(s, position)
                written[at, slot] = True
                assert np.array_equal(stored[at, :, slot], codes[r]), (name, s, i)
                if fmt != "bf16":
                    assert np.array_equal(stored_scales[at, :, slot], scales[r])
                want = bf16(codes[r].astype(np.float32) * scales[r][:, None])
                assert np.array_equal(got[r], want)
    for now, was in zip((c.keys, c.values, c.key_scales, c.value_scales), before):
        bits = lambda x: x.cpu().view(t.uint8).numpy().reshape(c.pages, kv_heads, page, -1)  # noqa: E731
        untouched = np.moveaxis(bits(now) == bits(was), 1, 2)[~written]
        assert untouched.all(), "slots of no row of the batch"


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_codes_are_those_of_the_exact_quotients(fmt):
    """Every mantissa of a row's largest value, at magnitudes from the smallest to the largest of bf16, under values of
    every mantissa: the ties among them (x 127 / m halfway between two codes) go to the even code."""
    rng = np.random.default_rng(16)
    exponents = [-133, -127, -120, -61, -60, -59, 0, 99, 100, 101, 120]
    rows = []
    for e in exponents:
        for mantissa in range(128, 256):
            x = np.ldexp(rng.integers(128, 256, 256).astype(np.float64), e - rng.integers(0, 12, 256))
            x = np.where(x <= mantissa * 2.0 ** e, x, 0) * rng.choice([-1, 1], 256)
            x[:3] = mantissa * 2.0 ** e, -mantissa * 2.0 ** (e - 1), mantissa * 2.0 ** (e - 2)
            rows.append(x)
    x = bf16(np.array(rows))
    c = Cache(rng, [(len(x), len(x))], 1, 256, 64, fmt)
    sq.kv_write(c.struct(), c.batch(), to_bf16(x), to_bf16(x))
    codes, scales = quantised(x[:, None], fmt)
    at = np.arange(len(x))
    for name in ("key", "value"):
        stored, by = getattr(c, name + "s").float().cpu().numpy(), getattr(c, name + "_scales").cpu().numpy()
        pages, slots = c.table[0, at // 64], at % 64
        assert np.array_equal(by[pages, :, slots], scales)
        assert np.array_equal(stored[pages, :, slots], codes)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_write_of_unbounded_rows(fmt):
    t = torch()
    rng = np.random.default_rng(5)
    c = Cache(rng, [(4, 20)], 2, 64, 16, fmt)
    k, v = c.new_rows(c.k), c.new_rows(c.v)
    k[0, 5], k[1, 64 + 9], v[2, 0] = np.inf, np.nan, -np.inf
    sq.kv_write(c.struct(), c.batch(), to_bf16(k), to_bf16(v))
    outs = [t.zeros((4, 128), dtype=t.bfloat16, device="cuda") for _ in range(2)]
    sq.kv_read(c.struct(), c.batch(), *outs)
    for out, bad in zip(outs, ({(0, 0), (1, 1)}, {(2, 0)})):
        got = from_bf16(out).reshape(4, 2, 64)
        for r in range(4):
            for h in range(2):
                assert np.isnan(got[r, h]).all() if (r, h) in bad else np.isfinite(got[r, h]).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,rotary,interleaved", [(128, 128, False), (64, 32, True), (80, 20, False), (256, 64, False)])
def test_write_with_rope(fmt, dim, rotary, interleaved):
    """Keys rotated on the way, and queries beside them, are the bits of sq_rope_add and a write of its output."""
    t = torch()
    rng = np.random.default_rng(dim)
    sizes = [(9, 700), (1, 1), (30, 30)]
    heads, kv_heads = 6, 2
    rope, _, _ = make_rope(rotary, interleaved)
    a, b = (Cache(np.random.default_rng(1), sizes, kv_heads, dim, 32, fmt, extra_rows=1) for _ in range(2))
    fused = to_bf16(bf16(rng.standard_normal((a.rows, (heads + 2 * kv_heads) * dim))))
    q, k, v = fused.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
    rotated = t.full((a.rows, heads * dim), 4.0, dtype=t.bfloat16, device="cuda")
    keep = fused.clone()
    sq.kv_write(a.struct(), a.batch(), k, v, rope=rope, queries=q, rotated=rotated)
    t.cuda.synchronize()
    assert t.equal(fused, keep)
    positions = np.concatenate([np.arange(n - r, n) for r, n in sizes] + [[0]]).astype(np.int32)
    p = t.from_numpy(positions).cuda()
    turned = t.empty((a.rows, (heads + kv_heads) * dim), dtype=t.bfloat16, device="cuda")
    sq.rope_add(rope, p, fused[:, :(heads + kv_heads) * dim], turned, dim)
    sq.kv_write(b.struct(), b.batch(), turned[:, heads * dim:], v)
    t.cuda.synchronize()
    assert t.equal(rotated[:-1], turned[:-1, :heads * dim]) and (rotated[-1] == 4).all()
    for x, y in ((a.keys, b.keys), (a.values, b.values), (a.key_scales, b.key_scales), (a.value_scales, b.value_scales)):
        assert t.equal(x.view(t.uint8), y.view(t.uint8))
    # Queries in place, keys alone.
    sq.kv_write(a.struct(), a.batch(), k, v, rope=rope, queries=q, rotated=q)
    sq.kv_write(b.struct(), b.batch(), keep[:, heads * dim:(heads + kv_heads) * dim], v, rope=rope)
    t.cuda.synchronize()
    assert t.equal(fused[:-1, :heads * dim], turned[:-1, :heads * dim])
    assert t.equal(a.keys.view(t.uint8), b.keys.view(t.uint8))


# ---------------------------------------------------------------- attention

def queries(rng, rows, heads, dim, size=1.5):
    return bf16(rng.standard_normal((rows, heads, dim)) * size)


RAGGED = [(1, 1), (1, 63), (0, 70), (1, 64), (3, 65), (0, 0), (1, 200), (2, 2), (1, 16), (4, 1000), (3, 1), (1, 0)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (1, 1, 16, 16), (8, 2, 64, 32), (10, 2, 128, 16), (7, 1, 128, 256), (24, 2, 80, 64), (16, 2, 256, 64), (6, 3, 144, 32),
    (64, 1, 128, 128),
])
def test_ragged_tokens(fmt, heads, kv_heads, dim, page):
    rng = np.random.default_rng(heads * dim + page)
    c = Cache(rng, RAGGED, kv_heads, dim, page, fmt, extra_rows=3).fill()
    q = queries(rng, c.rows, heads, dim)
    scale = 1 / math.sqrt(dim)
    want, bound = attention_f64(q, c, scale)
    got = run_attention(c, q, scale)
    check_attention(got[:c.live_rows], want, bound, fmt)
    assert np.all(got[c.live_rows:] == 123.0), "rows behind the last sequence"
    # The rows that see nothing: rows before position 0, and a sequence of no keys.
    assert np.all(got[c.starts[10]:c.starts[10] + 2] == 0.0) and np.all(got[c.starts[11]] == 0.0)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("causal,window", [(True, 1), (True, 5), (True, 64), (True, 130), (True, 5000), (False, 0)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (5, 1, 128), (4, 2, 192)])
def test_windows(fmt, causal, window, heads, kv_heads, dim):
    rng = np.random.default_rng(window + heads)
    c = Cache(rng, [(40, 333), (7, 7), (1, 500), (130, 131), (3, 2)], kv_heads, dim, 16, fmt).fill()
    q = queries(rng, c.rows, heads, dim)
    want, bound = attention_f64(q, c, 0.1, causal, window)
    check_attention(run_attention(c, q, 0.1, causal, window), want, bound, f"{fmt} {window}")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv_heads,dim,sizes", [
    (8, 1, 128, [(1, 20001)]),                      # one token, many parts of one unit
    (8, 8, 64, [(1, 9000), (1, 3), (1, 40000)]),
    (4, 1, 256, [(8, 7001), (8, 30)]),
    (12, 4, 128, [(8, 3333), (5, 12001), (8, 100)]),
    (4, 2, 128, [(300, 2900)]),
    (7, 1, 64, [(513, 513), (1, 1), (100, 4000)]),
    (2, 2, 256, [(200, 1200)]),
    (3, 1, 80, [(257, 700), (129, 129)]),
])
def test_long_and_chunks(fmt, heads, kv_heads, dim, sizes):
    rng = np.random.default_rng(dim + len(sizes))
    c = Cache(rng, sizes, kv_heads, dim, 64, fmt).fill()
    q = queries(rng, c.rows, heads, dim)
    scale = 1 / math.sqrt(dim)
    want, bound = attention_f64(q, c, scale)
    got = run_attention(c, q, scale)
    check_attention(got, want, bound, fmt)
    assert np.array_equal(got, run_attention(c, q, scale)), "a batch repeats its bits"
    # Another tile than the plan's usual one computes the same function.
    for chunk in (1, c.rows):
        check_attention(run_attention(c, q, scale, chunk=chunk), want, bound, f"{fmt} chunk {chunk}")


@pytest.mark.parametrize("size,scale", [(40.0, 1.0), (1e-3, 0.125), (3.0, -0.5), (1.0, 0.0)])
def test_score_ranges(size, scale):
    """Weights of one key alone (scores in the thousands), of all alike, negative and zero scales."""
    rng = np.random.default_rng(11)
    c = Cache(rng, [(6, 900), (1, 70)], 2, 128, 32, "bf16").fill()
    q = queries(rng, c.rows, 8, 128, size)
    want, bound = attention_f64(q, c, scale)
    check_attention(run_attention(c, q, scale), want, bound)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("sizes,chunk", [([(8, 300), (1, 40)], None), ([(200, 500), (3, 3)], None), ([(40, 40)], 1)])
def test_unseen_keys_touch_nothing(fmt, sizes, chunk):
    """New rows with NaN and infinite keys and values: the rows before them keep their bits; the rows that see them do
    what the formula does."""
    rng = np.random.default_rng(3)
    heads, dim = 4, 64
    clean = Cache(np.random.default_rng(8), sizes, 2, dim, 16, fmt).fill()
    bad = Cache(np.random.default_rng(8), sizes, 2, dim, 16, fmt)
    at = sizes[0][1] - 2                      # the last key but one of the first sequence
    bad.v[0][0, at, 3], bad.v[0][1, at, 60] = np.inf, np.nan
    bad.k[0][1, at + 1, 1] = np.nan
    bad.fill()
    q = queries(rng, clean.rows, heads, dim)
    a, b = (run_attention(c, q, 0.125, chunk=chunk) for c in (clean, bad))
    first = int(clean.starts[1]) - 2
    assert np.array_equal(a[:first], b[:first]) and np.array_equal(a[first + 2:], b[first + 2:])
    seen = b[first]
    if fmt == "bf16":
        assert np.all(seen[:2, 3] == np.inf) and np.isnan(seen[2:, 60]).all()
        assert np.array_equal(np.delete(seen[:2], 3, -1), np.delete(a[first, :2], 3, -1))
        assert np.array_equal(np.delete(seen[2:], 60, -1), np.delete(a[first, 2:], 60, -1))
    else:
        assert np.isnan(seen).all()           # the whole head row of the value reads back as NaN
    assert np.isnan(b[first + 1, 2:]).all(), "a NaN key makes its rows' scores NaN"


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kv_heads,dim", [(2, 64), (1, 128), (1, 256)])
def test_windows_over_unwritten_keys(fmt, kv_heads, dim):
    """Keys before every row's window that were never written: NaNs (also among the codes) and NaN scales."""
    t = torch()
    rng = np.random.default_rng(dim)
    window, sizes = 75, [(1, 700), (45, 900), (3, 80), (150, 333)]
    c = Cache(rng, sizes, kv_heads, dim, 32, fmt).fill()
    q = queries(rng, c.rows, 4, dim)
    want, bound = attention_f64(q, c, 0.1, True, window)
    for s, (n, keys) in enumerate(sizes):
        for position in range(max(0, keys - n - window + 1)):
            page, slot = c.slot(s, position)
            for x in (c.keys, c.values):
                x.view(t.uint8)[int(page), :, slot] = 0xFF
            for x in (c.key_scales, c.value_scales):
                x[int(page), :, slot] = math.nan
    for chunk in (1, c.rows):
        check_attention(run_attention(c, q, 0.1, True, window, chunk=chunk), want, bound, f"{fmt} chunk {chunk}")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [1, 70])
def test_holes(fmt, rows):
    """Page table entries that name no page: their keys are not seen, write nothing and read back as zeros."""
    t = torch()
    rng = np.random.default_rng(rows)
    c = Cache(rng, [(rows, 300), (1, 20)], 1, 64, 32, fmt).fill()
    c.table[0, 2], c.table[0, 8], c.table[1, 0] = c.pages, 0xFFFFFFFF, 0x80000000
    c.table_d.copy_(t.from_numpy(c.table.view(np.int32)))
    gone = lambda s, j: np.isin(j // 32, (2, 8) if s == 0 else (0,))  # noqa: E731
    q = queries(rng, c.rows, 3, 64)
    want, bound = attention_f64(q, c, 0.125, hidden=gone)
    got = run_attention(c, q, 0.125)
    check_attention(got, want, bound)
    assert np.all(got[-1] == 0.0)
    before = [x.clone() for x in (c.keys, c.values)]
    k = to_bf16(c.new_rows(c.k))
    sq.kv_write(c.struct(), c.batch(), k, k)
    out = t.ones((c.rows, 64), dtype=t.bfloat16, device="cuda")
    sq.kv_read(c.struct(), c.batch(), out)
    t.cuda.synchronize()
    for i in range(rows):
        hole = (300 - rows + i) // 32 in (2, 8)
        assert (out[i] == 0).all().item() == hole
    assert (out[-1] == 0).all()
    if rows == 1:
        for x, y in zip((c.keys, c.values), before):
            page = int(c.table[0, 9])
            same = x.view(t.uint8) == y.view(t.uint8)
            same[page] = True
            assert same.all()


def test_lengths_and_starts_out_of_range():
    """Lengths past the table count as all it holds; row starts past the rows, or falling, address nothing else."""
    t = torch()
    rng = np.random.default_rng(9)
    c = Cache(rng, [(2, 96)], 2, 64, 32, "bf16").fill()
    c.table = c.table[:, :3].copy()
    c.table_d = t.from_numpy(c.table.view(np.int32)).cuda()
    q = queries(rng, 2, 4, 64)
    want = run_attention(c, q, 0.125)
    c.lengths_d.fill_(-1)
    assert np.array_equal(run_attention(c, q, 0.125), want)
    c.starts_d.copy_(t.tensor([0, 2000000000], dtype=t.int32))
    assert np.array_equal(run_attention(c, q, 0.125), want)
    c.starts_d.copy_(t.tensor([2, 0], dtype=t.int32))
    assert np.all(run_attention(c, q, 0.125) == 123.0)
    rows = t.ones((2, 128), dtype=t.bfloat16, device="cuda")
    before = c.keys.clone()
    sq.kv_write(c.struct(), c.batch(), rows, rows)
    t.cuda.synchronize()
    assert t.equal(before.view(t.uint8), c.keys.view(t.uint8))


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_offsets_past_32_bits(fmt):
    """Pages from the far end of a cache of more than 2^32 bytes."""
    t = torch()
    rng = np.random.default_rng(4)
    heads, dim, page = 8, 128, 64
    c = Cache(rng, [(1, 500), (9, 200)], 2, dim, page, fmt).fill()
    want, bound = attention_f64(q := queries(rng, c.rows, heads, dim), c, 0.1)
    small = run_attention(c, q, 0.1)
    check_attention(small, want, bound)
    pages = (2 ** 32 + 2 ** 30) // (2 * page * dim * (2 if fmt == "bf16" else 1))
    shift = pages - c.pages
    for name in ("keys", "values", "key_scales", "value_scales"):
        x = getattr(c, name)
        far = t.zeros((pages, *x.shape[1:]), dtype=t.uint8 if fmt == "e4m3" and x.dim() == 4 else x.dtype, device="cuda")
        far[shift:] = x.view(far.dtype) if x.dim() == 4 else x
        setattr(c, name, far.view(x.dtype) if x.dim() == 4 else far)
    c.table = np.where(c.table < c.pages, c.table + shift, c.table).astype(np.uint32)
    c.table_d = t.from_numpy(c.table.view(np.int32)).cuda()
    c.pages = pages
    assert np.array_equal(run_attention(c, q, 0.1), small)
    k = to_bf16(c.new_rows(c.k))
    sq.kv_write(c.struct(), c.batch(), k, k)
    out = t.zeros_like(k)
    sq.kv_read(c.struct(), c.batch(), None, out)
    t.cuda.synchronize()
    codes, scales = quantised(c.new_rows(c.k).reshape(c.rows, 2, dim), fmt)
    assert np.array_equal(from_bf16(out), bf16(codes.astype(np.float32) * scales[..., None]).reshape(c.rows, -1))


def test_query_in_place_and_strided():
    t = torch()
    rng = np.random.default_rng(2)
    heads, dim = 6, 64
    c = Cache(rng, [(3, 700), (20, 90)], 2, dim, 16, "int8").fill()
    q = queries(rng, c.rows, heads, dim)
    want = run_attention(c, q, 0.125)
    fused = t.full((c.rows, heads * dim + 200), 3.0, dtype=t.bfloat16, device="cuda")
    fused[:, 96:96 + heads * dim] = to_bf16(q.reshape(c.rows, -1))
    view = fused[:, 96:96 + heads * dim]
    plan = sq.attention_plan(sq.AttentionShape(heads, c.shape, 1, 0, 0.125), 2, c.rows, 20)
    sq.attention_add(plan, c.struct(), c.batch(), view, view, sq.AttentionScratch(plan))
    t.cuda.synchronize()
    assert np.array_equal(from_bf16(view.contiguous()).reshape(want.shape), want)
    assert (fused[:, :96] == 3).all() and (fused[:, 96 + heads * dim:] == 3).all()


def test_graph_replays_with_other_lengths():
    """A captured step (rope and write, attention, read back) replayed over lengths and pages that change on the device
    between replays, with eager work in between: each replay is the eager result."""
    t = torch()
    rng = np.random.default_rng(6)
    heads, kv_heads, dim, page = 8, 2, 128, 32
    rope, _, _ = make_rope(128)
    c = Cache(rng, [(1, 2900), (1, 64), (1, 1500)], kv_heads, dim, page, "int8").fill()
    plan = sq.attention_plan(sq.AttentionShape(heads, c.shape, 1, 0, 0.09), 3, 3, 1)
    scratch, eager_scratch = sq.AttentionScratch(plan), sq.AttentionScratch(plan)
    fused = to_bf16(bf16(rng.standard_normal((3, (heads + 2 * kv_heads) * dim))))
    q, k, v = fused.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
    make = lambda w: t.zeros((3, w * dim), dtype=t.bfloat16, device="cuda")  # noqa: E731
    turned, out, back = make(heads), make(heads), make(kv_heads)

    def step(turned, out, back, scratch):
        sq.kv_write(c.struct(), c.batch(), k, v, rope=rope, queries=q, rotated=turned)
        sq.attention_add(plan, c.struct(), c.batch(), turned, out, scratch)
        sq.kv_read(c.struct(), c.batch(), back)

    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        step(turned, out, back, scratch)
    t.cuda.current_stream().wait_stream(side)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        step(turned, out, back, scratch)
    for lengths in ([2900, 64, 1500], [2901, 65, 1501], [1, 2, 3], [2912, 0, 700], [33, 64, 1504]):
        c.lengths_d.copy_(t.tensor(lengths, dtype=t.int32))
        fused.add_(0.25)
        graph.replay()
        t.cuda.synchronize()
        e = [make(heads), make(heads), make(kv_heads)]
        step(*e, eager_scratch)
        t.cuda.synchronize()
        for got, want in zip((turned, out, back), e):   # bits: keys that no step has written are NaN
            assert t.equal(got.view(t.int16), want.view(t.int16))


def test_graphs_that_share_a_workspace():
    """Two captured calls, of single tokens and of a chunk, over one workspace and in one stream, replayed in any order."""
    t = torch()
    rng = np.random.default_rng(15)
    parts = []
    for seed, sizes in ((1, [(1, 9000), (1, 77)]), (2, [(90, 4000), (1, 12)])):
        c = Cache(np.random.default_rng(seed), sizes, 2, 128, 64, "bf16").fill()
        q = queries(rng, c.rows, 8, 128)
        plan = sq.attention_plan(sq.AttentionShape(8, c.shape, 1, 0, 0.09), 2, c.rows, sizes[0][0])
        parts.append((c, plan, to_bf16(q.reshape(c.rows, -1)), run_attention(c, q, 0.09, plan=plan)))
    scratch = sq.AttentionScratch(max((plan for _, plan, *_ in parts), key=lambda plan: plan.partials))
    outs, graphs = [t.zeros_like(x) for _, _, x, _ in parts], []
    for (c, plan, x, _), out in zip(parts, outs):
        graphs.append(t.cuda.CUDAGraph())
        with t.cuda.graph(graphs[-1]):
            sq.attention_add(plan, c.struct(), c.batch(), x, out, scratch)
    for order in ((0, 1), (1, 0), (1, 1, 0), (0, 0, 1)):
        for out in outs:
            out.zero_()
        scratch.partials.fill_(-1)
        for i in order:
            graphs[i].replay()
        t.cuda.synchronize()
        for (*_, want), out in zip(parts, outs):
            assert np.array_equal(from_bf16(out).reshape(want.shape), want)


def test_binding_refuses_what_it_would_misread():
    t = torch()
    make = lambda *shape, dtype=t.int32: t.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    starts, lengths, table = make(2), make(1), make(1, 4)
    sq.kv_batch(starts, lengths, table, 1)
    for bad in ((make(2, dtype=t.int64), lengths, table), (starts, make(1, 2)[:, :1].expand(1, 2), make(2, 8)[:, :4]),
                (starts, lengths, make(4, 4).t()), (starts.cpu(), lengths, table)):
        with pytest.raises(ValueError):
            sq.kv_batch(*bad, 1)
    for bad in (make(2, 64, dtype=t.float16), make(64, 2, dtype=t.bfloat16).t(), make(2, 60, dtype=t.bfloat16),
                make(2, 64, dtype=t.float32), make(64, dtype=t.bfloat16)):
        with pytest.raises(ValueError):
            sq.head_rows(bad, 64)
    cache = Cache(np.random.default_rng(1), [(1, 5)], 2, 64, 16, "int8")
    with pytest.raises(ValueError):
        sq.kv_cache(cache.shape, cache.pages, cache.keys.transpose(1, 2), cache.values)
    with pytest.raises(ValueError):
        sq.kv_read(cache.struct(), cache.batch(), t.zeros((1, 128), dtype=t.bfloat16))


def test_two_streams_at_once():
    """Two batches on two streams, each with a workspace of its own."""
    t = torch()
    rng = np.random.default_rng(12)
    parts = []
    for seed, fmt in ((1, "bf16"), (2, "e4m3")):
        c = Cache(np.random.default_rng(seed), [(1, 6000), (4, 900)], 2, 128, 64, fmt).fill()
        q = queries(rng, c.rows, 8, 128)
        plan = sq.attention_plan(sq.AttentionShape(8, c.shape, 1, 0, 0.09), 2, c.rows, 4)
        parts.append((c, q, plan, sq.AttentionScratch(plan), run_attention(c, q, 0.09, plan=plan)))
    inputs = [to_bf16(q.reshape(len(q), -1)) for _, q, *_ in parts]
    outs = [t.zeros_like(x) for x in inputs]
    streams = [t.cuda.Stream() for _ in parts]
    t.cuda.synchronize()
    for _ in range(5):
        for (c, _, plan, scratch, _), x, out, stream in zip(parts, inputs, outs, streams):
            with t.cuda.stream(stream):
                sq.attention_add(plan, c.struct(), c.batch(), x, out, scratch)
    t.cuda.synchronize()
    for (*_, want), out in zip(parts, outs):
        assert np.array_equal(from_bf16(out).reshape(want.shape), want)


def test_many_sequences():
    """The most sequences a batch has, most of them short."""
    rng = np.random.default_rng(13)
    sizes = [(int(rng.random() < 0.8), int(rng.integers(0, 90))) for _ in range(1023)] + [(1, 3000)]
    c = Cache(rng, sizes, 1, 64, 16, "int8").fill()
    q = queries(rng, c.rows, 4, 64)
    want, bound = attention_f64(q, c, 0.125)
    check_attention(run_attention(c, q, 0.125), want, bound)


@pytest.mark.parametrize("units", [1, 8, 300])
def test_other_devices_plans(units):
    """Plans for fewer and more compute units: the same function on other shares."""
    rng = np.random.default_rng(14)
    c = Cache(rng, [(2, 3000), (1, 10), (60, 200)], 2, 64, 32, "bf16").fill()
    q = queries(rng, c.rows, 4, 64)
    want, bound = attention_f64(q, c, 0.125)
    plan = sq.attention_plan(sq.AttentionShape(4, c.shape, 1, 0, 0.125), 3, c.rows, 60, sq.Device(units))
    check_attention(run_attention(c, q, 0.125, plan=plan), want, bound)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [1, 100])
def test_between_the_projections(fmt, rows):
    """Norm, fused q|k|v projection, rope and cache write, attention, output projection onto the residual: the steps of
    a layer's first half in one stream. The cache and attention are checked from the bits the projection made, the
    output projection from the bits attention made."""
    from helpers import check_projection, make_weights, to_device, to_host
    t = torch()
    rng = np.random.default_rng(rows)
    hidden, heads, kv_heads, dim, past = 512, 8, 2, 64, 150
    rope, f, magnitude = make_rope(64)
    c = Cache(rng, [(rows, past + rows)], kv_heads, dim, 32, fmt).fill()
    w = make_weights(rng, sq.FMT_AF4G64, (heads + 2 * kv_heads) * dim, hidden)
    wo = make_weights(rng, sq.FMT_Q4K, hidden, heads * dim)
    first, last = sq.projection(w.segment()), sq.projection(wo.segment())
    work = sq.decode_workload if rows <= 32 else sq.prefill_workload
    p1 = sq.plan_for(work(w.n, hidden, rows), first)
    p2 = sq.plan_for(work(hidden, wo.k, rows, sq.EPILOGUE_RESIDUAL), last)
    from splash_q4 import synthetic
    x_bits = synthetic.bf16_bits(rng.standard_normal((p1.storage_rows, hidden)).astype(np.float32))
    ones = to_device(synthetic.bf16_bits(np.ones(hidden, np.float32)))
    x = to_device(x_bits)
    made = lambda r, width: t.zeros((r, width), dtype=t.bfloat16, device="cuda")  # noqa: E731
    normal, fused = made(p1.storage_rows, hidden), made(p1.storage_rows, w.n)
    attended, out = made(p2.storage_rows, heads * dim), made(p2.storage_rows, hidden)
    s1, s2 = sq.Scratch(p1), sq.Scratch(p2)
    plan = sq.attention_plan(sq.AttentionShape(heads, c.shape, 1, 0, 0.125), 1, rows, rows)
    scratch = sq.AttentionScratch(plan)
    q, k, v = fused[:rows].split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
    sq.call("sq_norm_add_rms", sq.stream_handle(), sq.view(x), sq.byref(sq.NormWeights(sq.view(ones), 0)),
            sq.view(normal), hidden, rows, None, sq.LINEAR_INPUT_PLAIN, None)
    sq.linear_add(p1, first, normal, fused, scratch=s1.struct())
    raw = fused.clone()
    sq.kv_write(c.struct(), c.batch(), k, v, rope=rope, queries=q, rotated=q)
    sq.attention_add(plan, c.struct(), c.batch(), q, attended[:rows], scratch)
    sq.linear_add(p2, last, attended, out, residual=x, scratch=s2.struct())
    t.cuda.synchronize()
    rows_of = from_bf16(raw[:rows]).reshape(rows, -1, dim)
    positions = np.arange(past, past + rows)
    turned, scale = rope_f64(rows_of[:, :heads + kv_heads], positions, f, magnitude, False)
    got_q = from_bf16(fused[:rows]).reshape(rows, -1, dim)[:, :heads]
    assert np.all(np.abs(got_q - turned[:, :heads]) <= rope_bound(turned, scale)[:, :heads])
    # The keys as the library rotated them: its own rope's bits (held to the definition above).
    p = t.from_numpy(positions.astype(np.int32)).cuda()
    keys = t.empty((rows, kv_heads * dim), dtype=t.bfloat16, device="cuda")
    sq.rope_add(rope, p, raw[:rows, heads * dim:(heads + kv_heads) * dim], keys, dim)
    c.k[0][:, past:] = np.moveaxis(from_bf16(keys).reshape(rows, kv_heads, dim), 1, 0)
    c.v[0][:, past:] = np.moveaxis(rows_of[:, heads + kv_heads:], 1, 0)
    want, bound = attention_f64(got_q, c, 0.125)
    a = from_bf16(attended[:rows]).reshape(rows, heads, dim)
    check_attention(a, want, bound, "attention of the projected rows")
    bits = to_host(attended[:rows].view(t.int16), np.uint16)
    check_projection(to_host(out[:rows].view(t.int16), np.uint16), bits, wo, "output projection",
                     residual=x_bits[:rows])
