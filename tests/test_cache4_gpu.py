"""The paged cache in 4 bits through the C ABI against its definition in 64 bits: codes and scales at every border, rows of
odd sizes, NaN and infinity where somebody looks and where nobody does, and attention over its pages on every tile."""
import math

import numpy as np
import pytest

import splash_q4 as sq
from attention_oracle import attention_f64, bf16, check_attention, from_bf16, run_attention, to_bf16, torch
from cache4_oracle import Cache4, packed, quantised4, scale_bytes, values4
from test_attention_weights import attend

pytestmark = pytest.mark.gpu

SIZES = [(3, 3), (0, 40), (1, 100), (0, 0), (17, 50), (2, 33), (5, 3)]   # the last has rows before position 0
DIMS = [32, 64, 96, 128, 160, 256]


@pytest.mark.parametrize("kv_heads,dim,page", [(1, 32, 16), (3, 64, 32), (2, 96, 16), (8, 128, 16), (5, 160, 128), (2, 256, 1024)])
def test_write_and_read(kv_heads, dim, page):
    t = torch()
    rng = np.random.default_rng(dim + page)
    c = Cache4(rng, SIZES, kv_heads, dim, page, extra_rows=2)
    for part, value in ((c.k, 1e-37), (c.v, 3e38)):     # magnitudes at both ends, and a row of zeros
        part[4][0, 40] = bf16(np.clip(part[4][0, 40] * value / 4, -3.3e38, 3.3e38))
        part[4][0, 41] = 0.0
    k, v = c.new_rows(c.k), c.new_rows(c.v)
    width = kv_heads * dim
    fused = t.zeros((c.rows, 2 * width + 8), dtype=t.bfloat16, device="cuda")
    fused[:, :width], fused[:, width + 8:] = to_bf16(k), to_bf16(v)
    before = [x.clone() for x in (c.keys, c.values, c.key_scales, c.value_scales)]
    sq.kv_write(c.struct(), c.batch(), fused[:, :width], fused[:, width + 8:])
    outs = [t.full((c.rows, width), 7.0, dtype=t.bfloat16, device="cuda") for _ in range(2)]
    sq.kv_read(c.struct(), c.batch(), *outs)
    t.cuda.synchronize()
    written = np.zeros((c.pages, page), bool)
    for name, rows, out in (("key", k, outs[0]), ("value", v, outs[1])):
        codes, scales = quantised4(rows.reshape(c.rows, kv_heads, dim))
        stored, by = getattr(c, name + "s").cpu().numpy(), getattr(c, name + "_scales").cpu().numpy()
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
                assert np.array_equal(stored[at, :, slot], packed(codes[r])), (name, s, i)
                assert np.array_equal(by[at, :, slot], scales[r]), (name, s, i)
                assert np.array_equal(got[r], values4(codes[r], scales[r]))
    for now, was in zip((c.keys, c.values, c.key_scales, c.value_scales), before):
        same = np.moveaxis((now == was).cpu().numpy(), 1, 2)[~written]
        assert same.all(), "slots of no row of the batch"


def test_codes_at_every_border():
    """Every bf16 mantissa for a group's largest value, at exponents from the least to the largest, over values of every
    mantissa down to a hundredth of it: borders between codes, and between scales, are among them."""
    rng = np.random.default_rng(16)
    rows = []
    for e in (-133, -128, -127, -126, -125, -60, 0, 1, 77, 118, 119, 120):
        for mantissa in range(128, 256):
            x = np.ldexp(rng.integers(128, 256, 256).astype(np.float64), e - rng.integers(0, 8, 256))
            x = np.where(x <= mantissa * 2.0 ** e, x, 0) * rng.choice([-1, 1], 256)
            x[:3] = mantissa * 2.0 ** e, -mantissa * 2.0 ** (e - 1), mantissa * 2.0 ** (e - 2)
            x[32:64:5] = -mantissa * 2.0 ** e
            rows.append(x)
    x = bf16(np.array(rows))
    c = Cache4(rng, [(len(x), len(x))], 1, 256, 64)
    sq.kv_write(c.struct(), c.batch(), to_bf16(x), to_bf16(x))
    out = torch().zeros((len(x), 256), dtype=torch().bfloat16, device="cuda")
    sq.kv_read(c.struct(), c.batch(), out)
    codes, scales = quantised4(x[:, None])
    at = np.arange(len(x))
    pages, slots = c.table[0, at // 64], at % 64
    assert np.array_equal(c.key_scales.cpu().numpy()[pages, :, slots], scales)
    assert np.array_equal(c.values.cpu().numpy()[pages, :, slots], packed(codes))
    want = values4(codes, scales)[:, 0]
    assert np.array_equal(from_bf16(out), want)
    # No value is off by more than one of its group's scale (but for those past the largest scale's range).
    step = np.ldexp(1.0, scales[:, 0].astype(int) - 127).repeat(32, -1)
    assert np.all((np.abs(want - x) <= step) | (np.abs(x) > 7 * 2.0 ** 125))


def test_write_of_unbounded_rows():
    t = torch()
    rng = np.random.default_rng(5)
    c = Cache4(rng, [(4, 20)], 2, 64, 16)
    k, v = c.new_rows(c.k), c.new_rows(c.v)
    k[0, 5], k[1, 64 + 39], v[2, 0] = np.inf, np.nan, -np.inf
    sq.kv_write(c.struct(), c.batch(), to_bf16(k), to_bf16(v))
    outs = [t.zeros((4, 128), dtype=t.bfloat16, device="cuda") for _ in range(2)]
    sq.kv_read(c.struct(), c.batch(), *outs)
    for out, bad in zip(outs, ({(0, 0), (1, 3)}, {(2, 0)})):
        got = from_bf16(out).reshape(4, 4, 32)          # [rows, groups]
        for r in range(4):
            for g in range(4):
                assert np.isnan(got[r, g]).all() if (r, g) in bad else np.isfinite(got[r, g]).all()


@pytest.mark.parametrize("rows", [2500, 40])
def test_write_with_rope_is_rope_and_write(rows):
    """Many rows (a wave each) and few (a workgroup each), keys rotated on the way and queries beside them."""
    t = torch()
    rng = np.random.default_rng(rows)
    sizes, heads, kv_heads, dim = [(rows - 7, rows + 11), (7, 7)], 6, 2, 96
    rope = sq.RotaryPositions(sq.RopeConfig(rotary_dim=48, layout=sq.ROPE_HALF, scaling=0, base=1e4))
    a, b = (Cache4(np.random.default_rng(1), sizes, kv_heads, dim, 32) for _ in range(2))
    fused = to_bf16(bf16(rng.standard_normal((a.rows, (heads + 2 * kv_heads) * dim))))
    q, k, v = fused.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
    rotated = t.zeros((a.rows, heads * dim), dtype=t.bfloat16, device="cuda")
    sq.kv_write(a.struct(), a.batch(), k, v, rope=rope, queries=q, rotated=rotated)
    p = t.from_numpy(np.concatenate([np.arange(n - r, n) for r, n in sizes]).astype(np.int32)).cuda()
    turned = t.empty((a.rows, (heads + kv_heads) * dim), dtype=t.bfloat16, device="cuda")
    sq.rope_add(rope, p, fused[:, :(heads + kv_heads) * dim], turned, dim)
    sq.kv_write(b.struct(), b.batch(), turned[:, heads * dim:], v)
    t.cuda.synchronize()
    assert t.equal(rotated, turned[:, :heads * dim])
    for x, y in ((a.keys, b.keys), (a.values, b.values), (a.key_scales, b.key_scales), (a.value_scales, b.value_scales)):
        assert t.equal(x, y)


# ---------------------------------------------------------------- attention

def queries(rng, rows, heads, dim, size=1.5):
    return bf16(rng.standard_normal((rows, heads, dim)) * size)


RAGGED = [(1, 1), (1, 63), (0, 70), (1, 64), (3, 65), (0, 0), (1, 200), (2, 2), (1, 16), (4, 1000), (3, 1), (1, 0)]


@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (1, 1, 32, 16), (8, 2, 64, 32), (10, 2, 128, 16), (7, 1, 128, 256), (24, 2, 96, 64), (16, 2, 256, 64), (6, 3, 160, 32),
    (64, 1, 128, 128),
])
def test_ragged_tokens(heads, kv_heads, dim, page):
    rng = np.random.default_rng(heads * dim + page)
    c = Cache4(rng, RAGGED, kv_heads, dim, page, extra_rows=3).fill()
    q = queries(rng, c.rows, heads, dim)
    scale = 1 / math.sqrt(dim)
    want, bound = attention_f64(q, c, scale)
    got = run_attention(c, q, scale)
    check_attention(got[:c.live_rows], want, bound)
    assert np.all(got[c.live_rows:] == 123.0), "rows behind the last sequence"
    assert np.all(got[c.starts[10]:c.starts[10] + 2] == 0.0) and np.all(got[c.starts[11]] == 0.0)


@pytest.mark.parametrize("causal,window", [(True, 1), (True, 5), (True, 64), (True, 130), (True, 5000), (False, 0)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (5, 1, 128), (4, 2, 192)])
def test_windows(causal, window, heads, kv_heads, dim):
    rng = np.random.default_rng(window + heads)
    c = Cache4(rng, [(40, 333), (7, 7), (1, 500), (130, 131), (3, 2)], kv_heads, dim, 16).fill()
    q = queries(rng, c.rows, heads, dim)
    want, bound = attention_f64(q, c, 0.1, causal, window)
    check_attention(run_attention(c, q, 0.1, causal, window), want, bound)


@pytest.mark.parametrize("heads,kv_heads,dim,sizes", [
    (8, 1, 128, [(1, 20001)]), (8, 8, 64, [(1, 9000), (1, 3), (1, 40000)]), (4, 1, 256, [(8, 7001), (8, 30)]),
    (12, 4, 128, [(8, 3333), (5, 12001), (8, 100)]), (4, 2, 128, [(300, 2900)]), (7, 1, 64, [(513, 513), (1, 1), (100, 4000)]),
    (2, 2, 256, [(200, 1200)]), (3, 1, 96, [(257, 700), (129, 129)]), (3, 1, 32, [(65, 700)]),
])
def test_long_and_chunks(heads, kv_heads, dim, sizes):
    rng = np.random.default_rng(dim + len(sizes))
    c = Cache4(rng, sizes, kv_heads, dim, 64).fill()
    q = queries(rng, c.rows, heads, dim)
    scale = 1 / math.sqrt(dim)
    want, bound = attention_f64(q, c, scale)
    got = run_attention(c, q, scale)
    check_attention(got, want, bound)
    assert np.array_equal(got, run_attention(c, q, scale)), "a batch repeats its bits"
    for chunk in (1, c.rows):
        check_attention(run_attention(c, q, scale, chunk=chunk), want, bound, f"chunk {chunk}")


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("sizes,chunk", [([(8, 300), (1, 40)], None), ([(200, 500), (3, 3)], None), ([(40, 40)], 1)])
def test_unseen_keys_touch_nothing(dim, sizes, chunk):
    """New rows with NaN and infinite keys and values: the rows before them keep their bits, and in those that see them a
    value's group is NaN and its other groups what they were."""
    rng = np.random.default_rng(3)
    heads = 4
    clean = Cache4(np.random.default_rng(8), sizes, 2, dim, 16).fill()
    bad = Cache4(np.random.default_rng(8), sizes, 2, dim, 16)
    at = sizes[0][1] - 2                      # the last key but one of the first sequence
    bad.v[0][0, at, 3], bad.v[0][1, at, 60] = np.inf, np.nan
    bad.k[0][1, at + 1, 1] = np.nan
    bad.fill()
    q = queries(rng, clean.rows, heads, dim)
    a, b = (run_attention(c, q, 0.125, chunk=chunk) for c in (clean, bad))
    first = int(clean.starts[1]) - 2
    assert np.array_equal(a[:first], b[:first]) and np.array_equal(a[first + 2:], b[first + 2:])
    seen = b[first].reshape(heads, -1, 32)
    assert np.isnan(seen[:2, 0]).all() and np.isnan(seen[2:, 1]).all()
    assert np.array_equal(seen[:2, 1:], a[first].reshape(heads, -1, 32)[:2, 1:])
    assert np.array_equal(seen[2:, 0], a[first].reshape(heads, -1, 32)[2:, 0])
    assert np.isnan(b[first + 1, 2:]).all(), "a NaN key makes its rows' scores NaN"


@pytest.mark.parametrize("byte,code,want", [(253, 2, 2.0 ** 126), (253, 6, math.inf), (254, 0, 0.0), (254, 5, math.inf),
                                            (254, 13, -math.inf), (255, 0, math.nan), (1, 2, 2.0 ** -126)])
@pytest.mark.parametrize("chunk", [1, 60])
def test_scale_bytes_of_no_write(byte, code, want, chunk):
    """Bytes that another program left: a page's value that one row of the batch sees alone, read back and attended to."""
    t = torch()
    rng = np.random.default_rng(9)
    c = Cache4(rng, [(60, 60)], 1, 128, 16).fill()
    page, slot = c.slot(0, 59)
    base = run_attention(c, q := queries(rng, 60, 2, 128), 0.1, chunk=chunk)
    c.values[int(page), 0, slot] = 0
    c.values[int(page), 0, slot, 20] = code          # value 40, of group 1
    c.value_scales[int(page), 0, slot, 1] = byte
    back = t.zeros((60, 128), dtype=t.bfloat16, device="cuda")
    sq.kv_read(c.struct(), c.batch(), None, back)
    assert np.array_equal(from_bf16(back)[59, 40], want, equal_nan=True)
    got = run_attention(c, q, 0.1, chunk=chunk)
    assert np.array_equal(got[:59], base[:59])
    if math.isnan(want):
        assert np.isnan(got[59, :, 32:64]).all() and np.isfinite(got[59, :, :32]).all()
    elif math.isinf(want):
        assert np.all(got[59, :, 40] == want) and np.isfinite(np.delete(got[59], 40, -1)).all()
    else:
        assert np.isfinite(got[59]).all()


@pytest.mark.parametrize("byte", [253, 254])
@pytest.mark.parametrize("heads,kv_heads,dim,tile", [(8, 1, 64, 16), (16, 2, 96, 16), (8, 1, 128, 16), (24, 1, 128, 32), (20, 1, 64, 32),
                                                     (8, 1, 256, 16)])
def test_finite_values_under_scale_bytes_of_no_write(byte, heads, kv_heads, dim, tile):
    """The largest finite values that another program's bytes make, which some rows of a tile see and others do not, within the
    bound of all weights of few rows: two bf16 each. (Weights are alike, so that none takes a sum past fp32's range.)"""
    t = torch()
    rng = np.random.default_rng(byte + dim)
    sizes, scale = [(3, 60), (1, 33), (2, 700)], 0.01
    c = Cache4(rng, sizes, kv_heads, dim, 16).fill()
    held = [c.stored(s) for s in range(len(sizes))]
    for s, (n, keys) in enumerate(sizes):
        for position in range(keys - n, keys):
            page, slot = c.slot(s, position)
            codes = rng.choice(np.array([0, 1, 2, 9, 10] if byte == 253 else [0, 1, 9], np.uint8), (kv_heads, 32))
            c.values[int(page), :, slot, 16:32] = t.from_numpy(packed(codes)).cuda()      # group 1
            c.value_scales[int(page), :, slot, 1] = byte
            held[s][1][:, position, 32:64] = np.where(codes & 8, -0.5, 0.5) * (codes & 7) * 2.0 ** (byte - 127)
    q = queries(rng, c.rows, heads, dim)
    plan = sq.attention_plan(sq.AttentionShape(heads, c.shape, 1, 0, scale), len(sizes), c.rows, 1)
    assert plan.tile_rows == tile
    got, group = run_attention(c, q, scale, plan=plan), heads // kv_heads
    for s, (n, keys) in enumerate(sizes):
        for i in range(n):
            for h in range(kv_heads):
                k, v = (x[h, :keys - n + i + 1] for x in held[s])
                rows = slice(h * group, (h + 1) * group)
                want, bound = attend(q[c.starts[s] + i, rows], k, v, scale)
                err = np.abs(got[c.starts[s] + i, rows] - want)
                assert np.all(err <= bound), (s, i, h, np.max(err / bound))


@pytest.mark.parametrize("kv_heads,dim", [(2, 64), (1, 96), (1, 128), (1, 256)])
def test_windows_over_unwritten_keys(kv_heads, dim):
    t = torch()
    rng = np.random.default_rng(dim)
    window, sizes = 75, [(1, 700), (45, 900), (3, 80), (150, 333)]
    c = Cache4(rng, sizes, kv_heads, dim, 32).fill()
    q = queries(rng, c.rows, 4, dim)
    want, bound = attention_f64(q, c, 0.1, True, window)
    for s, (n, keys) in enumerate(sizes):
        for position in range(max(0, keys - n - window + 1)):
            page, slot = c.slot(s, position)
            for x in (c.keys, c.values, c.key_scales, c.value_scales):
                x[int(page), :, slot] = 0xFF
    for chunk in (1, c.rows):
        check_attention(run_attention(c, q, 0.1, True, window, chunk=chunk), want, bound, f"chunk {chunk}")


@pytest.mark.parametrize("rows", [1, 70])
def test_holes(rows):
    t = torch()
    rng = np.random.default_rng(rows)
    c = Cache4(rng, [(rows, 300), (1, 20)], 1, 64, 32).fill()
    c.table[0, 2], c.table[0, 8], c.table[1, 0] = c.pages, 0xFFFFFFFF, 0x80000000
    c.table_d.copy_(t.from_numpy(c.table.view(np.int32)))
    gone = lambda s, j: np.isin(j // 32, (2, 8) if s == 0 else (0,))  # noqa: E731
    q = queries(rng, c.rows, 3, 64)
    want, bound = attention_f64(q, c, 0.125, hidden=gone)
    got = run_attention(c, q, 0.125)
    check_attention(got, want, bound)
    assert np.all(got[-1] == 0.0)
    out = t.ones((c.rows, 64), dtype=t.bfloat16, device="cuda")
    k = to_bf16(c.new_rows(c.k))
    sq.kv_write(c.struct(), c.batch(), k, k)
    sq.kv_read(c.struct(), c.batch(), out)
    for i in range(rows):
        assert (out[i] == 0).all().item() == ((300 - rows + i) // 32 in (2, 8))
    assert (out[-1] == 0).all()


def test_offsets_past_32_bits():
    """Pages from the far end of a cache of more than 2^32 bytes of codes."""
    t = torch()
    rng = np.random.default_rng(4)
    heads, dim, page = 8, 128, 64
    c = Cache4(rng, [(1, 500), (9, 200)], 2, dim, page).fill()
    q = queries(rng, c.rows, heads, dim)
    small = run_attention(c, q, 0.1)
    pages = (2 ** 32 + 2 ** 30) // (page * dim)
    shift = pages - c.pages
    for name in ("keys", "values", "key_scales", "value_scales"):
        x = getattr(c, name)
        far = t.zeros((pages, *x.shape[1:]), dtype=t.uint8, device="cuda")
        far[shift:] = x
        setattr(c, name, far)
    c.table = np.where(c.table < c.pages, c.table + shift, c.table).astype(np.uint32)
    c.table_d = t.from_numpy(c.table.view(np.int32)).cuda()
    c.pages = pages
    assert np.array_equal(run_attention(c, q, 0.1), small)
    k = c.new_rows(c.k)
    sq.kv_write(c.struct(), c.batch(), to_bf16(k), to_bf16(k))
    out = t.zeros((c.rows, 2 * dim), dtype=t.bfloat16, device="cuda")
    sq.kv_read(c.struct(), c.batch(), None, out)
    assert np.array_equal(from_bf16(out), values4(*quantised4(k.reshape(c.rows, 2, dim))).reshape(c.rows, -1))


def test_graph_replays_with_other_lengths():
    """A captured step (rope and write, attention, read back) over lengths that change on the device between replays."""
    t = torch()
    rng = np.random.default_rng(6)
    heads, kv_heads, dim, page = 8, 2, 128, 32
    rope = sq.RotaryPositions(sq.RopeConfig(rotary_dim=128, layout=sq.ROPE_HALF, scaling=0, base=1e4))
    c = Cache4(rng, [(1, 2900), (1, 64), (1, 1500)], kv_heads, dim, page).fill()
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
    for lengths in ([2900, 64, 1500], [2901, 65, 1501], [1, 2, 3], [2912, 0, 700]):
        c.lengths_d.copy_(t.tensor(lengths, dtype=t.int32))
        fused.add_(0.25)
        graph.replay()
        t.cuda.synchronize()
        e = [make(heads), make(heads), make(kv_heads)]
        step(*e, eager_scratch)
        t.cuda.synchronize()
        for got, want in zip((turned, out, back), e):
            assert t.equal(got.view(t.int16), want.view(t.int16))


def test_scale_bytes_of_head_sizes():
    for dim in DIMS:
        assert sq.kv_cache_size(sq.KvShape(3, dim, 16, sq.KV_E2M1), 5).key_scales == 5 * 3 * 16 * scale_bytes(dim)
