"""Attention with capped and biased scores, first keys and prefixes through the C ABI against its definition in 64 bits: every
format and tile, caps from below the scores to far above them, ragged batches with rows that see nothing, packed documents
over one stored sequence, NaN and infinity where nobody looks, graphs."""
import math

import numpy as np
import pytest

import splash_q4 as sq
from attention_oracle import FORMATS, Cache, bf16, check_attention, from_bf16, run_attention, to_bf16, torch
from cache4_oracle import Cache4
from scores_oracle import device_words, run_scored, scored_f64, scores_of

pytestmark = pytest.mark.gpu

ALL = [*FORMATS, "e2m1"]


def make(rng, sizes, kv_heads, dim, page, fmt, **kw):
    if fmt == "e2m1":
        return Cache4(rng, sizes, kv_heads, dim, page, **kw)
    return Cache(rng, sizes, kv_heads, dim, page, fmt, **kw)


def queries(rng, rows, heads, dim, size=1.5):
    return bf16(rng.standard_normal((rows, heads, dim)) * size)


def slopes_of(heads):
    return [2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)]


def check(c, q, scale, chunks=(None,), what="", causal=True, window=0, **kw):
    want, bound = scored_f64(q, c, scale, causal, window, **kw)
    for chunk in chunks:
        got = run_scored(c, q, scale, causal, window, chunk, **kw)
        check_attention(got[:c.live_rows], want, bound, f"{what} chunk {chunk}")
        assert np.all(got[c.live_rows:] == 123.0), "rows behind the last sequence"
    return want


@pytest.mark.parametrize("fmt", ALL)
@pytest.mark.parametrize("cap", [0.5, 30.0, 127.0, 129.0, 1e5])
@pytest.mark.parametrize("size", [1.5, 40.0])
def test_caps(fmt, cap, size):
    """Scores far below the cap, about it and far above it."""
    rng = np.random.default_rng(int(cap))
    c = make(rng, [(6, 700), (1, 70), (40, 90)], 2, 128, 32, fmt).fill()
    q = queries(rng, c.rows, 8, 128, size)
    check(c, q, 0.3, (1, 40), f"{fmt} {cap}", cap=cap)


@pytest.mark.parametrize("scale", [0.125, -0.5, 0.0])
def test_caps_of_other_scales(scale):
    rng = np.random.default_rng(3)
    c = make(rng, [(6, 300), (1, 70)], 2, 64, 32, "bf16").fill()
    check(c, queries(rng, c.rows, 4, 64), scale, (1, 7), cap=20.0)


RAGGED = [(1, 1), (1, 63), (0, 70), (1, 64), (3, 65), (0, 0), (1, 200), (2, 2), (1, 16), (4, 1000), (3, 1), (1, 0)]


@pytest.mark.parametrize("fmt", ALL)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 64, 32), (10, 2, 128, 16), (16, 2, 256, 64), (24, 2, 96, 64),
                                                     (7, 1, 160, 128), (64, 1, 128, 16)])
def test_ragged_tokens(fmt, heads, kv_heads, dim, page):
    rng = np.random.default_rng(heads * dim + page)
    c = make(rng, RAGGED, kv_heads, dim, page, fmt, extra_rows=3).fill()
    q = queries(rng, c.rows, heads, dim)
    n = len(RAGGED)
    begins, prefixes = np.array([0, 60, 0, 63, 64, 0, 7, 5, 17, 990, 0, 3]), np.array([0, 9, 0, 64, 65, 0, 4, 1, 99, 996, 1, 0])
    assert len(begins) == len(prefixes) == n
    for kw in (dict(cap=25.0), dict(slopes=slopes_of(heads)), dict(begins=begins), dict(prefixes=prefixes),
               dict(cap=25.0, slopes=slopes_of(heads), begins=begins, prefixes=prefixes)):
        want = check(c, q, 1 / math.sqrt(dim), (None, c.rows), f"{fmt} {list(kw)}", **kw)
    # Rows that see nothing: before position 0, of no keys, and behind their sequence's begin.
    got = run_scored(c, q, 0.1, begins=begins, prefixes=prefixes)
    assert np.all(got[c.starts[10]:c.starts[10] + 2] == 0.0) and np.all(got[c.starts[11]] == 0.0)
    assert np.all(got[c.starts[8]] == 0.0) and np.all(want[c.starts[8]] == 0.0)


@pytest.mark.parametrize("fmt", ALL)
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 1), (True, 70), (True, 500), (False, 0)])
def test_masks_of_chunks(fmt, causal, window):
    """Begins and prefixes on, before and behind tiles' and units' edges, under windows and without causality."""
    rng = np.random.default_rng(window)
    sizes = [(200, 900), (64, 64), (130, 131), (1, 500), (70, 700), (5, 3), (33, 640)]
    c = make(rng, sizes, 2, 64, 16, fmt).fill()
    q = queries(rng, c.rows, 6, 64)
    for begins, prefixes in (([0, 1, 64, 499, 0, 0, 640], None), ([700, 63, 65, 500, 690, 2, 607], None),
                             ([2 ** 31, 2 ** 32 - 1, 131, 501, 699, 3, 639], None),
                             (None, [0, 64, 128, 2 ** 32 - 1, 640, 3, 639]), (None, [800, 1, 131, 200, 2 ** 31, 1, 0]),
                             ([64, 32, 127, 0, 300, 1, 600], [850, 40, 100, 500, 666, 2, 640])):
        if prefixes is not None and not causal:
            continue
        check(c, q, 0.1, (None, 1), f"{fmt} {begins} {prefixes}", causal, window, begins=begins, prefixes=prefixes)


@pytest.mark.parametrize("fmt", ALL)
@pytest.mark.parametrize("heads,kv_heads,dim,sizes,causal", [
    (8, 1, 128, [(1, 20001)], True), (8, 8, 64, [(1, 9000), (1, 3), (1, 40000)], True), (4, 1, 256, [(8, 7001), (8, 30)], True),
    (4, 2, 128, [(300, 2900)], True), (2, 2, 256, [(200, 1200)], True), (3, 1, 96, [(257, 700), (129, 129)], False),
    (33, 1, 128, [(1, 3000)], True),
])
def test_slopes_over_long_contexts(fmt, heads, kv_heads, dim, sizes, causal):
    """Slopes from a half to 2^-8, one negative (scores that grow with the distance) and one zero."""
    rng = np.random.default_rng(dim + len(sizes))
    c = make(rng, sizes, kv_heads, dim, 64, fmt).fill()
    q = queries(rng, c.rows, heads, dim)
    slopes = slopes_of(heads)
    slopes[-1] = -0.01
    if heads > 2:
        slopes[1] = 0.0
    check(c, q, 1 / math.sqrt(dim), (None, 1, c.rows), fmt, causal, slopes=slopes)
    a, b = (run_scored(c, q, 0.1, causal, slopes=slopes, cap=20.0) for _ in range(2))
    assert np.array_equal(a, b), "a batch repeats its bits"


@pytest.mark.parametrize("fmt", ALL)
@pytest.mark.parametrize("chunk", [None, 1])
def test_packed_documents(fmt, chunk):
    """Documents of one stored sequence, each a sequence of the batch with a begin and the same pages, are the documents stored
    each for itself, and a question behind them sees all."""
    rng = np.random.default_rng(31)
    heads, kv_heads, dim, page = 6, 2, 64, 16
    ends = [5, 70, 71, 200, 333, 400]
    whole = make(rng, [(400, 400)], kv_heads, dim, page, fmt).fill()
    q = queries(rng, 400, heads, dim)
    begins = [0, *ends[:-2], 0]                    # the last one is the question
    first = [0, *ends[:-1]]
    packed = make(np.random.default_rng(1), [(e - f, e) for f, e in zip(first, ends)], kv_heads, dim, page, fmt)
    packed.k, packed.v = [[part[0][:, :e] for e in ends] for part in (whole.k, whole.v)]
    for name in ("keys", "values", "key_scales", "value_scales"):
        setattr(packed, name, getattr(whole, name))
    packed.pages = whole.pages
    packed.table = np.repeat(whole.table, len(ends), 0)
    packed.table_d = torch().from_numpy(packed.table.view(np.int32)).cuda()
    for kw in (dict(), dict(slopes=slopes_of(heads), cap=30.0)):
        check(packed, q, 0.125, (chunk,), fmt, begins=begins, **kw)
    got = run_scored(packed, q, 0.125, chunk=chunk, begins=begins)
    for s, (f, e) in enumerate(zip(first, ends)):
        if begins[s] != f:
            continue
        alone = make(np.random.default_rng(2), [(e - f, e - f)], kv_heads, dim, page, fmt)
        alone.k, alone.v = [[part[0][:, f:e]] for part in (whole.k, whole.v)]
        want, bound = scored_f64(q[f:e], alone.fill(), 0.125)
        check_attention(got[f:e], want, bound, f"document {s}")


@pytest.mark.parametrize("fmt", ALL)
@pytest.mark.parametrize("chunk", [None, 1])
def test_hidden_keys_touch_nothing(fmt, chunk):
    """NaN in every form a page can hold it, infinities and NaN scales, before the begins and behind the prefixes."""
    t = torch()
    rng = np.random.default_rng(8)
    sizes = [(40, 300), (1, 200), (100, 500), (8, 77)]
    begins, prefixes = [250, 150, 130, 70], [290, 0, 450, 77]
    c = make(rng, sizes, 2, 128, 16, fmt).fill()
    q = queries(rng, c.rows, 4, 128)
    what = dict(cap=30.0, slopes=slopes_of(4), begins=begins, prefixes=prefixes)
    want, bound = scored_f64(q, c, 0.1, **what)
    clean = run_scored(c, q, 0.1, chunk=chunk, **what)
    for s, (n, keys) in enumerate(sizes):
        for position in range(begins[s]):
            page, slot = c.slot(s, position)
            for x in (c.keys, c.values):
                x.view(t.uint8)[int(page), :, slot] = 0xFF
            for x in (c.key_scales, c.value_scales):
                x.view(t.uint8)[int(page), :, slot] = 0xFF
    got = run_scored(c, q, 0.1, chunk=chunk, **what)
    check_attention(got, want, bound, fmt)
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("chunk", [None, 1])
def test_infinite_scores_under_a_cap(chunk):
    """A key whose product is infinite has the cap for its score; a NaN stays one."""
    rng = np.random.default_rng(2)
    c = Cache(rng, [(3, 40)], 1, 64, 16, "bf16")
    c.k[0][0, 7] = 0.0
    c.k[0][0, 7, 3] = np.inf
    c.k[0][0, 39, 3] = np.nan
    q = queries(rng, 3, 2, 64)
    q[:, 0, 3], q[:, 1, 3] = 1.0, -1.0
    c.fill()
    got = run_scored(c, q, 0.1, chunk=chunk, cap=5.0)
    c.k[0][0, 7, 3], c.k[0][0, 39, 3] = 9984.0, 0.0       # scores of 1000 have the cap all the same
    want, bound = scored_f64(q, c, 0.1, cap=5.0)
    # q.k with an infinity times zeros is NaN: the other values of that key are zero, so its products 0 q are fine.
    check_attention(got[:2], want[:2], bound[:2])
    assert np.isnan(got[2]).all()


@pytest.mark.parametrize("fmt", ALL)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("cap", [30.0, 400.0])
@pytest.mark.parametrize("chunk", [None, 1])
def test_hidden_keys_touch_nothing_under_a_cap_alone(fmt, dim, cap, chunk):
    """The same for calls that have a cap and no slopes (a kernel of their own where rows are many and the cap is not above 128):
    NaN in keys, values and scales before the begins and behind the prefixes."""
    t = torch()
    rng = np.random.default_rng(dim)
    sizes = [(130, 400), (1, 200), (100, 500), (64, 77)]
    begins, prefixes = [250, 150, 130, 70], [290, 0, 450, 77]
    c = make(rng, sizes, 2, dim, 16, fmt).fill()
    q = queries(rng, c.rows, 4, dim)
    what = dict(cap=cap, begins=begins, prefixes=prefixes)
    want, bound = scored_f64(q, c, 0.1, **what)
    clean = run_scored(c, q, 0.1, chunk=chunk, **what)
    for s in range(len(sizes)):
        for position in range(begins[s]):
            page, slot = c.slot(s, position)
            for x in (c.keys, c.values, c.key_scales, c.value_scales):
                x.view(t.uint8)[int(page), :, slot] = 0xFF
    got = run_scored(c, q, 0.1, chunk=chunk, **what)
    check_attention(got, want, bound, fmt)
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("fmt", ALL)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("cap", [5.0, 60.0, 300.0])
@pytest.mark.parametrize("chunk", [None, 1])
def test_unbounded_scores_that_all_rows_see(fmt, dim, cap, chunk):
    """Products that overflow, in a tile that all rows see: their scores are the cap, or below zero. (One key has a value where
    the queries are large and nothing else there; the other keys' scores are far within the cap or not.) A key that is NaN makes the
    outputs of its head NaN, whichever tile it lies in, and no others."""
    rng = np.random.default_rng(dim + int(cap))
    c = make(rng, [(140, 400)], 2, dim, 16, fmt)
    for part in c.k:
        part[:, :, 3] = 0.0
        part[:, 70] = 0.0
        part[:, 70, 3] = 1e30
    q = queries(rng, c.rows, 4, dim, 0.3)
    q[:, ::2, 3], q[:, 1::2, 3] = 1e30, -1e30
    got = run_scored(c.fill(), bf16(q), 0.05, chunk=chunk, cap=cap)
    # In 64 bits by products of 20 caps, of which the hyperbolic tangent is one to 2^-56.
    for part in c.k:
        part[:, 70, 3] = bf16(400.0 * cap)
    q[:, ::2, 3], q[:, 1::2, 3] = 1.0, -1.0
    want, bound = scored_f64(q, c, 0.05, cap=cap)
    check_attention(got, want, bound, fmt)
    c.k[0][1, 200, 5] = np.nan
    nan = run_scored(c.fill(), q, 0.05, chunk=chunk, cap=cap)
    assert np.isnan(nan[:, 2:]).all() and np.isfinite(nan[:, :2]).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("chunk", [None, 1])
def test_unbounded_values_under_a_cap_alone(dim, chunk):
    """Infinite and NaN values that some rows of a tile see: those rows have them, and the others keep their bits."""
    rng = np.random.default_rng(dim)
    c = make(rng, [(140, 400)], 2, dim, 16, "bf16").fill()
    q = queries(rng, c.rows, 4, dim)
    clean = run_scored(c, q, 0.05, chunk=chunk, cap=30.0)
    c.v[0][0, 300, 7], c.v[0][1, 390, 40] = np.inf, np.nan
    got = run_scored(c.fill(), q, 0.05, chunk=chunk, cap=30.0)
    at = np.arange(260, 400)
    want = clean.copy()
    want[at >= 300, :2, 7] = np.inf
    want[at >= 390, 2:, 40] = np.nan
    assert np.array_equal(got, want, equal_nan=True)


def test_nothing_to_do_is_the_plain_call():
    """No part given: the bits of the plain call; neutral parts: its function."""
    rng = np.random.default_rng(4)
    for sizes, chunk in (([(1, 900), (3, 70)], None), ([(100, 900), (3, 70)], None)):
        c = make(rng, sizes, 2, 64, 16, "int8").fill()
        q = queries(rng, c.rows, 8, 64)
        plain = run_attention(c, q, 0.1)
        assert np.array_equal(run_scored(c, q, 0.1), plain)
        want, bound = scored_f64(q, c, 0.1)
        for kw in (dict(slopes=[0.0] * 8), dict(begins=[0, 0]), dict(prefixes=[0, 0]), dict(cap=1e30)):
            check_attention(run_scored(c, q, 0.1, chunk=chunk, **kw), want, bound, str(kw))


def test_many_sequences():
    rng = np.random.default_rng(13)
    sizes = [(int(rng.integers(0, 4)), int(rng.integers(0, 90))) for _ in range(1023)] + [(1, 3000)]
    c = make(rng, sizes, 1, 64, 16, "bf16").fill()
    begins, prefixes = rng.integers(0, 60, 1024), rng.integers(0, 100, 1024)
    check(c, queries(rng, c.rows, 4, 64), 0.125, (None, 40), begins=begins, prefixes=prefixes, slopes=slopes_of(4), cap=10.0)


@pytest.mark.parametrize("units", [1, 3, 8, 40])
@pytest.mark.parametrize("fmt", ["bf16", "e2m1"])
def test_units_dealt_whole(fmt, units):
    """Batches whose units nearly fill a small device's workgroups, alike and of many lengths, so that they stay whole in one turn,
    in several, or are cut: the same function, and the same bits each time."""
    rng = np.random.default_rng(units)
    t = torch()
    for sizes, chunk in (([(1, 300 + 7 * i) for i in range(24)], 1), ([(1, int(n)) for n in rng.integers(1, 700, 70)], 1),
                         ([(64 + 3 * i, 64 + 3 * i) for i in range(9)], 64), ([(500, 900)], 500), ([(1, 10)] * 300, 1),
                         ([(int(n), int(n) + 30) for n in rng.integers(0, 130, 25)], 100)):
        c = make(rng, sizes, 2, 64, 16, fmt).fill()
        q = queries(rng, c.rows, 4, 64)
        begins = [int(rng.integers(0, k // 2 + 1)) for _, k in sizes]
        want, bound = scored_f64(q, c, 0.125, begins=begins, cap=20.0)
        scores, keep = scores_of(cap=20.0, begins=begins)
        plan = sq.attention_plan(sq.AttentionShape(4, c.shape, 1, 0, 0.125), len(sizes), c.rows, min(chunk, c.rows),
                                 sq.Device(units))
        outs = []
        for _ in range(2):
            out, scratch = t.zeros((c.rows, 256), dtype=t.bfloat16, device="cuda"), sq.AttentionScratch(plan)
            scratch.partials.fill_(0xFF)
            sq.attention_add(plan, c.struct(), c.batch(), to_bf16(q.reshape(c.rows, -1)), out, scratch, scores=scores)
            outs.append(from_bf16(out).reshape(q.shape))
        check_attention(outs[0], want, bound, f"{len(sizes)} sequences")
        assert np.array_equal(*outs)
        del keep


@pytest.mark.parametrize("kv_heads", [1, 3, 5, 8])
@pytest.mark.parametrize("window,prefix", [(0, 0), (90, 0), (0, 150), (70, 130)])
def test_whole_units_of_uneven_heads(kv_heads, window, prefix):
    """Units kept whole whose key heads do not divide the eight dies' workgroups, and whose lengths do not grow with the row."""
    rng = np.random.default_rng(kv_heads + window)
    t = torch()
    for sizes, chunk, units in (([(1, 200 + 9 * i) for i in range(40)], 1, 16), ([(150 + 11 * i, 170 + 13 * i) for i in range(8)], 300, 24),
                                ([(int(n), int(n) + 3) for n in rng.integers(0, 200, 30)], 200, 256)):
        c = make(rng, sizes, kv_heads, 64, 16, "bf16").fill()
        heads = 2 * kv_heads
        q = queries(rng, c.rows, heads, 64)
        prefixes = [prefix] * len(sizes)
        want, bound = scored_f64(q, c, 0.125, window=window, prefixes=prefixes, slopes=slopes_of(heads))
        scores, keep = scores_of(prefixes=prefixes, slopes=slopes_of(heads))
        plan = sq.attention_plan(sq.AttentionShape(heads, c.shape, 1, window, 0.125), len(sizes), c.rows, min(chunk, c.rows),
                                 sq.Device(units))
        out, scratch = t.full((c.rows, heads * 64), 123.0, dtype=t.bfloat16, device="cuda"), sq.AttentionScratch(plan)
        scratch.partials.fill_(0xFF)
        sq.attention_add(plan, c.struct(), c.batch(), to_bf16(q.reshape(c.rows, -1)), out, scratch, scores=scores)
        check_attention(from_bf16(out).reshape(q.shape)[:c.live_rows], want, bound, f"{len(sizes)} sequences")
        del keep


def test_holes_under_a_prefix():
    t = torch()
    rng = np.random.default_rng(6)
    for rows in (1, 70):
        c = make(rng, [(rows, 300), (1, 20)], 1, 64, 32, "e4m3").fill()
        q = queries(rng, c.rows, 3, 64)
        c.table[0, 2], c.table[1, 0] = c.pages, 0x80000000
        c.table_d.copy_(t.from_numpy(c.table.view(np.int32)))
        got = run_scored(c, q, 0.125, prefixes=[300, 20], slopes=[0.1, 0.2, 0.0])
        # The hole's keys out of the way: the definition over the others, their distances kept.
        c.k[0], c.v[0] = c.k[0].copy(), c.v[0].copy()
        bias = [0.1, 0.2, 0.0]
        k, v = c.stored(0)
        j = np.array([x for x in range(300) if x // 32 != 2])
        for i in range(rows):
            for h in range(3):
                s = q[i, h] @ k[0][j].T * 0.125 - bias[h] * np.abs(300 - rows + i - j)
                w = np.exp(s - s.max())
                want = w @ v[0][j] / w.sum()
                assert np.all(np.abs(got[i, h] - want) <= 2 ** -7 * (w @ np.abs(v[0][j]) / w.sum()) * 1.1)
        assert np.all(got[-1] == 0.0)


def test_query_in_place():
    rng = np.random.default_rng(2)
    t = torch()
    c = make(rng, [(3, 700), (20, 90)], 2, 64, 16, "int8").fill()
    q = queries(rng, c.rows, 6, 64)
    want = run_scored(c, q, 0.125, cap=15.0)
    fused = t.full((c.rows, 6 * 64 + 200), 3.0, dtype=t.bfloat16, device="cuda")
    fused[:, 96:96 + 384] = to_bf16(q.reshape(c.rows, -1))
    plan = sq.attention_plan(sq.AttentionShape(6, c.shape, 1, 0, 0.125), 2, c.rows, 20)
    scores, _ = scores_of(cap=15.0)
    view = fused[:, 96:96 + 384]
    sq.attention_add(plan, c.struct(), c.batch(), view, view, sq.AttentionScratch(plan), scores=scores)
    t.cuda.synchronize()
    assert np.array_equal(from_bf16(view.contiguous()).reshape(want.shape), want)
    assert (fused[:, :96] == 3).all() and (fused[:, 96 + 384:] == 3).all()


@pytest.mark.parametrize("rows", [1, 60])
def test_graph_replays_with_other_scores(rows):
    """A captured call over slopes, begins, prefixes and lengths that change on the device between replays."""
    t = torch()
    rng = np.random.default_rng(7)
    c = make(rng, [(rows, 2900), (1, 64), (rows, 1500)], 2, 128, 32, "e4m3").fill()
    q = to_bf16(queries(rng, c.rows, 8, 128).reshape(c.rows, -1))
    plan = sq.attention_plan(sq.AttentionShape(8, c.shape, 1, 0, 0.09), 3, c.rows, rows)
    scratch, other = sq.AttentionScratch(plan), sq.AttentionScratch(plan)
    scores, (slopes, begins, prefixes) = scores_of(20.0, slopes_of(8), [0, 0, 0], [0, 0, 0])
    out, eager = t.zeros_like(q), t.zeros_like(q)
    run = lambda to, s: sq.attention_add(plan, c.struct(), c.batch(), q, to, s, scores=scores)  # noqa: E731
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        run(out, scratch)
    t.cuda.current_stream().wait_stream(side)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        run(out, scratch)
    for i, lengths in enumerate(([2900, 64, 1500], [2800, 60, 70], [100, 1, 1400])):
        c.lengths_d.copy_(t.tensor(lengths, dtype=t.int32))
        slopes.mul_(0.5)
        begins.copy_(device_words([10 * i, 5, 90 * i]))
        prefixes.copy_(device_words([2900, 0, 1450 - i]))
        out.zero_()
        graph.replay()
        t.cuda.synchronize()
        run(eager, other)
        t.cuda.synchronize()
        assert t.equal(out.view(t.int16), eager.view(t.int16))


def test_two_streams_at_once():
    t = torch()
    rng = np.random.default_rng(12)
    parts = []
    for seed, fmt, kw in ((1, "bf16", dict(cap=30.0)), (2, "e2m1", dict(slopes=slopes_of(8)))):
        c = make(np.random.default_rng(seed), [(1, 6000), (4, 900)], 2, 128, 64, fmt).fill()
        q = queries(rng, c.rows, 8, 128)
        plan = sq.attention_plan(sq.AttentionShape(8, c.shape, 1, 0, 0.09), 2, c.rows, 4)
        parts.append((c, to_bf16(q.reshape(c.rows, -1)), plan, sq.AttentionScratch(plan), scores_of(**kw),
                      run_scored(c, q, 0.09, **kw)))
    outs, streams = [t.zeros_like(x) for _, x, *_ in parts], [t.cuda.Stream() for _ in parts]
    t.cuda.synchronize()
    for _ in range(5):
        for (c, x, plan, scratch, (scores, _), _), out, stream in zip(parts, outs, streams):
            with t.cuda.stream(stream):
                sq.attention_add(plan, c.struct(), c.batch(), x, out, scratch, scores=scores)
    t.cuda.synchronize()
    for (*_, want), out in zip(parts, outs):
        assert np.array_equal(from_bf16(out).reshape(want.shape), want)
