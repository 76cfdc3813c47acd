"""Rotary positions, the paged cache and attention on the host: the rope's frequencies against their formulas, the
cache's and plan's sizes, and every refusal of the entry points, all before anything is launched (the views point
nowhere)."""
import ctypes
import math

import pytest

import splash_q4 as sq


def config(**kw):
    d = dict(rotary_dim=128, layout=sq.ROPE_HALF, scaling=sq.ROPE_SCALING_NONE, base=1e4, factor=8.0,
             original_positions=8192)
    return sq.RopeConfig(**{**d, **kw})


def test_rope_frequencies():
    f, magnitude = sq.rope_frequencies(config(rotary_dim=6))
    assert magnitude == 1.0
    assert f == pytest.approx([1.0, 1e4 ** (-1 / 3), 1e4 ** (-2 / 3)], rel=1e-14)
    f, _ = sq.rope_frequencies(config(rotary_dim=6, scaling=sq.ROPE_SCALING_LINEAR))
    assert f == pytest.approx([1 / 8, 1e4 ** (-1 / 3) / 8, 1e4 ** (-2 / 3) / 8], rel=1e-14)
    f, _ = sq.rope_frequencies(config(rotary_dim=6, scaling=sq.ROPE_SCALING_NTK))
    # The slowest pair of the scaled base turns factor times slower, the first as fast as before.
    assert f[0] == 1.0 and f[2] == pytest.approx(1e4 ** (-2 / 3) / 8, rel=1e-13)


def test_rope_yarn():
    plain, _ = sq.rope_frequencies(config())
    f, magnitude = sq.rope_frequencies(config(scaling=sq.ROPE_SCALING_YARN))
    assert magnitude == pytest.approx(0.1 * math.log(8) + 1, rel=2 ** -24)
    turns = [8192 * x / (2 * math.pi) for x in plain]
    for x, y, t in zip(plain, f, turns):
        assert x / 8 * (1 - 1e-12) <= y <= x * (1 + 1e-12)
        if t > 34:          # past the rounded-outwards bounds of 32 turns and 1
            assert y == x
        if t < 0.85:
            assert y == pytest.approx(x / 8, rel=1e-14)
    assert any(x / 8 < y * (1 - 1e-3) < x * (1 - 2e-3) for x, y in zip(plain, f)), "the ramp between them"
    assert f == sorted(f, reverse=True)


def test_rope_wavelength():
    plain, _ = sq.rope_frequencies(config(base=5e5))
    f, magnitude = sq.rope_frequencies(config(base=5e5, scaling=sq.ROPE_SCALING_WAVELENGTH))
    assert magnitude == 1.0
    for x, y in zip(plain, f):
        w = 2 * math.pi / x
        if w < 8192 / 4:
            want = x
        elif w > 8192:
            want = x / 8
        else:
            t = (8192 / w - 1) / 3
            want = (1 - t) * x / 8 + t * x
        assert y == pytest.approx(want, rel=1e-13)


@pytest.mark.parametrize("change,message", [
    (dict(rotary_dim=0), "even number"), (dict(rotary_dim=7), "even number"), (dict(rotary_dim=258), "even number"),
    (dict(layout=2), "layout"), (dict(scaling=5), "scaling"), (dict(base=1.0), "base"), (dict(base=math.nan), "base"),
    (dict(scaling=1, factor=0.5), "factor"), (dict(scaling=1, factor=math.inf), "factor"),
    (dict(scaling=2, rotary_dim=2), "one pair"), (dict(scaling=3, original_positions=0), "original"),
    (dict(scaling=4, low=4.0, high=2.0), "bound"), (dict(scaling=3, low=-1.0), "bound"),
])
def test_rope_config_refusals(change, message):
    with pytest.raises(sq.InvalidArgument, match=message):
        sq.rope_frequencies(config(**change))


def buffer(nbytes, at=1 << 20):
    return sq.Buffer(at, nbytes)


def rows_of(rows, heads, dim, stride=None, at=1 << 20, short=0):
    stride = stride or heads * dim
    return sq.HeadRows(buffer(2 * ((rows - 1) * stride + heads * dim) - short, at), heads, stride)


def refused(name, message, *args):
    with pytest.raises(sq.InvalidArgument, match=message):
        sq.call(name, None, *args)


def test_rope_refusals():
    by = ctypes.byref
    rope = sq.Rope(64, sq.ROPE_HALF, 1.0, buffer(256))
    x, positions = rows_of(3, 4, 128), buffer(12)

    def no(message, rope=rope, positions=positions, rows=3, dim=128, x=x, y=None):
        refused("sq_rope_add", message, by(rope), positions, rows, dim, by(x), by(y if y is not None else x))

    no("multiple of 16", dim=120)
    no("multiple of 16", dim=272)
    no("even number", rope=sq.Rope(130, 0, 1.0, buffer(4096)))
    no("layout", rope=sq.Rope(64, 2, 1.0, buffer(256)))
    no("magnitude", rope=sq.Rope(64, 0, math.inf, buffer(256)))
    no("frequencies", rope=sq.Rope(64, 0, 1.0, buffer(255)))
    no("8-byte", rope=sq.Rope(64, 0, 1.0, buffer(256, (1 << 20) + 4)))
    no("positions", positions=buffer(11))
    no("4-byte", positions=buffer(12, (1 << 20) + 2))
    no("2\\^20", rows=(1 << 20) + 1)
    no("same heads", y=rows_of(3, 5, 128))
    no("row stride", x=rows_of(3, 4, 128, 516))
    no("row stride", x=sq.HeadRows(buffer(1 << 16), 4, 504))
    no("holds", x=rows_of(3, 4, 128, short=1))
    no("16-byte", x=rows_of(3, 4, 128, at=(1 << 20) + 8))
    no("null", x=sq.HeadRows(sq.Buffer(None, 1 << 16), 4, 512))
    no("in place", y=rows_of(3, 4, 128, 520))
    refused("sq_rope_add", "null", None, positions, 3, 128, by(x), by(x))
    # No rows: nothing to launch, and nothing is looked at.
    sq.call("sq_rope_add", None, by(rope), sq.Buffer(None, 0), 0, 128, by(x), by(x))


def kv_shape(**kw):
    return sq.KvShape(**{**dict(kv_heads=2, head_dim=64, page_rows=32, format=sq.KV_INT8), **kw})


def cache(pages=10, at=None, short=None, **kw):
    shape = kv_shape(**kw)
    size = sq.kv_cache_size(shape, pages)
    names = ("keys", "values", "key_scales", "value_scales")
    views = [buffer(getattr(size, n) - (short == n), (1 << 20) + (4 if at == n else 0)) for n in names]
    return sq.KvCache(shape, pages, *views)


def batch(sequences=3, rows=5, pages=4, **kw):
    d = dict(row_starts=buffer(4 * sequences + 4), lengths=buffer(4 * sequences),
             page_table=buffer(4 * sequences * pages))
    d.update(kw)
    return sq.KvBatch(sequences, rows, pages, d["row_starts"], d["lengths"], d["page_table"])


def test_cache_sizes():
    size = sq.kv_cache_size(kv_shape(), 10)
    assert (size.keys, size.values, size.key_scales, size.value_scales) == (40960, 40960, 2560, 2560)
    size = sq.kv_cache_size(kv_shape(format=sq.KV_BF16), 10)
    assert (size.keys, size.values, size.key_scales, size.value_scales) == (81920, 81920, 0, 0)
    # Offsets past 32 bits: a cache of 2^40 bytes.
    assert sq.kv_cache_size(kv_shape(kv_heads=8, head_dim=128, page_rows=1024), 1 << 20).keys == 1 << 40


@pytest.mark.parametrize("change,message", [
    (dict(kv_heads=0), "key heads"), (dict(kv_heads=1025), "key heads"), (dict(head_dim=0), "multiple of 16"),
    (dict(head_dim=72), "multiple of 16"), (dict(head_dim=272), "multiple of 16"), (dict(page_rows=8), "pages"),
    (dict(page_rows=48), "pages"), (dict(page_rows=2048), "pages"), (dict(format=3), "format"),
])
def test_cache_shape_refusals(change, message):
    with pytest.raises(sq.InvalidArgument, match=message):
        sq.kv_cache_size(kv_shape(**change), 4)
    with pytest.raises(sq.InvalidArgument, match="has pages"):
        sq.kv_cache_size(kv_shape(), 0)


CACHE_REFUSALS = [
    ("cache keys", dict(short="keys"), {}), ("cache values", dict(short="values"), {}),
    ("key scales", dict(short="key_scales"), {}), ("value scales", dict(short="value_scales"), {}),
    ("16-byte", dict(at="keys"), {}), ("16-byte", dict(at="value_scales"), {}),
    ("sequences", {}, dict(sequences=0)), ("sequences", {}, dict(sequences=1025)),
    ("2\\^20 rows", {}, dict(rows=(1 << 20) + 1)), ("pages", {}, dict(pages=0)),
    ("2\\^30 keys", {}, dict(pages=(1 << 25) + 1)), ("row starts", {}, dict(row_starts=buffer(15))),
    ("lengths", {}, dict(lengths=buffer(11))), ("page table", {}, dict(page_table=buffer(47))),
    ("4-byte", {}, dict(lengths=buffer(12, (1 << 20) + 1))),
]


@pytest.mark.parametrize("message,c,b", CACHE_REFUSALS)
def test_cache_and_batch_refusals(message, c, b):
    by = ctypes.byref
    k, out = rows_of(5, 2, 64), rows_of(5, 4, 64)
    refused("sq_kv_add_write", message, by(cache(**c)), by(batch(**b)), by(k), by(k), None, None, None)
    refused("sq_kv_add_read", message, by(cache(**c)), by(batch(**b)), by(k), by(k))
    plan = attention_plan(rows=5, sequences=3)
    buffers = sq.AttentionBuffers(out, out, buffer(plan.partials))
    refused("sq_attention_add", message, by(buffers), by(cache(**c)), by(batch(**b)), by(plan))


def test_write_and_read_refusals():
    by = ctypes.byref
    c, b, k = cache(), batch(), rows_of(5, 2, 64)
    rope = sq.Rope(64, sq.ROPE_HALF, 1.0, buffer(256))
    q = rows_of(5, 8, 64)
    refused("sq_kv_add_write", "key heads", by(c), by(b), by(rows_of(5, 3, 64)), by(k), None, None, None)
    refused("sq_kv_add_write", "value rows", by(c), by(b), by(k), by(rows_of(5, 2, 64, short=2)), None, None, None)
    refused("sq_kv_add_write", "with a rope", by(c), by(b), by(k), by(k), None, by(q), by(q))
    refused("sq_kv_add_write", "with a rope", by(c), by(b), by(k), by(k), by(rope), by(q), None)
    refused("sq_kv_add_write", "even number", by(c), by(b), by(k), by(k), by(sq.Rope(66, 0, 1.0, buffer(512))), None,
            None)
    refused("sq_kv_add_write", "same heads", by(c), by(b), by(k), by(k), by(rope), by(q), by(rows_of(5, 6, 64)))
    refused("sq_kv_add_read", "key heads", by(c), by(b), by(k), by(rows_of(5, 4, 64)))
    for name in ("cache", "batch", "key rows"):
        args = [by(c), by(b), by(k)]
        args[("cache", "batch", "key rows").index(name)] = None
        refused("sq_kv_add_write", f"{name} is null", *args, by(k), None, None, None)
    # No rows, or neither keys nor values to read: nothing to launch.
    sq.call("sq_kv_add_write", None, by(c), by(batch(rows=0)), by(k), by(k), None, None, None)
    sq.call("sq_kv_add_read", None, by(c), by(batch(rows=0)), by(k), by(k))
    sq.call("sq_kv_add_read", None, by(c), by(b), None, None)


def attention_shape(heads=4, causal=1, window=0, scale=0.125, **kw):
    return sq.AttentionShape(heads, kv_shape(**kw), causal, window, scale)


def attention_plan(shape=None, sequences=3, rows=5, chunk=1, dev=None):
    return sq.attention_plan(shape or attention_shape(), sequences, rows, chunk, dev)


def test_attention_plans():
    few = {(128, sq.KV_BF16): 32, (128, sq.KV_INT8): 32, (64, sq.KV_E4M3): 32, (256, sq.KV_BF16): 16, (256, sq.KV_INT8): 16}
    for heads, kv_heads, chunk in ((32, 8, 1), (32, 8, 4), (40, 8, 8), (34, 2, 1), (64, 1, 1), (33, 1, 1), (8, 8, 100)):
        for (dim, format), most in few.items():
            shape = attention_shape(heads=heads, kv_heads=kv_heads, head_dim=dim, format=format)
            plan = sq.attention_plan(shape, 4, 400, chunk)
            packed = heads // kv_heads * chunk
            # The smallest tile that holds a sequence's new rows with their query heads.
            assert plan.tile_rows == next((t for t in (16, 32) if packed <= t <= most), 128)
            assert plan.workgroups % 8 == 0 and plan.partials > 16 * plan.workgroups
    small = attention_plan(dev=sq.Device(10))
    assert small.workgroups % 8 == 0 and 10 <= small.workgroups < 32
    with pytest.raises(sq.InvalidArgument, match="65536 compute units"):
        attention_plan(dev=sq.Device(65537))
    # The work of a call is counted in 52 bits, row starts that overlap included.
    kv, huge, by = kv_shape(kv_heads=1024, head_dim=16, page_rows=1024, format=sq.KV_BF16), buffer(1 << 62), ctypes.byref
    plan = sq.attention_plan(sq.AttentionShape(1024, kv, 1, 0, 0.25), 1024, 1 << 14, 1)
    rows = sq.HeadRows(huge, 1024, 1024 * 16)
    refused("sq_attention_add", "less than 2", by(sq.AttentionBuffers(rows, rows, huge)),
            by(sq.KvCache(kv, 1 << 20, huge, huge, sq.Buffer(0, 0), sq.Buffer(0, 0))),
            by(sq.KvBatch(1024, 1 << 14, 1 << 9, huge, huge, huge)), by(plan))


@pytest.mark.parametrize("shape,sizes,message", [
    (dict(heads=0), {}, "multiple of the key heads"), (dict(heads=5), {}, "multiple of the key heads"),
    (dict(heads=130), {}, "at most 64"), (dict(causal=0, window=4), {}, "window"), (dict(causal=2), {}, "causal"),
    (dict(scale=math.inf), {}, "scale"), (dict(scale=math.nan), {}, "scale"), (dict(page_rows=24), {}, "pages"),
    ({}, dict(sequences=0), "sequences"), ({}, dict(sequences=1025), "sequences"), ({}, dict(rows=0), "rows"),
    ({}, dict(rows=(1 << 20) + 1), "rows"), ({}, dict(chunk=0), "new rows"), ({}, dict(chunk=6), "new rows"),
])
def test_attention_plan_refusals(shape, sizes, message):
    with pytest.raises(sq.InvalidArgument, match=message):
        attention_plan(attention_shape(**shape), **sizes)


def test_attention_refusals():
    by = ctypes.byref
    plan, q = attention_plan(), rows_of(5, 4, 64)
    good = dict(query=q, output=q, partials=buffer(plan.partials))

    def no(message, plan=plan, cache=cache(), batch=batch(), **kw):
        b = sq.AttentionBuffers(*[{**good, **kw}[n] for n in ("query", "output", "partials")])
        refused("sq_attention_add", message, by(b), by(cache), by(batch), by(plan))

    no("another cache", cache=cache(page_rows=64))
    no("another cache", cache=cache(format=sq.KV_E4M3))
    no("larger than its", batch=batch(sequences=4))
    no("larger than its", batch=batch(rows=6))
    no("heads", query=rows_of(5, 6, 64))
    no("heads", output=rows_of(5, 2, 64))
    no("query rows", query=rows_of(5, 4, 64, short=1))
    no("output rows", output=rows_of(5, 4, 64, short=1))
    no("in place", output=rows_of(5, 4, 64, 264))
    no("attention partials", partials=buffer(plan.partials - 1))
    no("16-byte", partials=buffer(plan.partials, (1 << 20) + 8))
    for field in ("tile_rows", "waves", "workgroups", "partials"):
        wrong = sq.AttentionPlan.from_buffer_copy(plan)
        setattr(wrong, field, getattr(wrong, field) + 8)
        no("fields", plan=wrong)
    none = sq.AttentionBuffers(*[good[n] for n in ("query", "output", "partials")])
    sq.call("sq_attention_add", None, by(none), by(cache()), by(batch(rows=0)), by(plan))


def test_head_rows_of_tensors():
    torch = pytest.importorskip("torch")
    fused = torch.zeros((3, 768), dtype=torch.bfloat16)
    v = sq.head_rows(fused[:, 512:], 64)
    assert (v.heads, v.row_stride, v.buffer.bytes) == (4, 768, 2 * (2 * 768 + 256))
    for bad in (fused.t(), fused[:, :100], fused.float(), fused[:, ::2]):
        with pytest.raises(ValueError, match="head rows"):
            sq.head_rows(bad, 64)


def test_cxx_face(tmp_path):
    """The C++ header compiles against the library; its sizes are the C ABI's, its refusals exceptions."""
    import pathlib
    import shutil
    import subprocess
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    exe, libs = tmp_path / "attention_check", sq.LIBRARY.parent
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(sq.HEADER.parent),
                    str(pathlib.Path(__file__).parent / "cxx_attention_check.cpp"), "-L", str(libs), "-lsplash_q4",
                    f"-Wl,-rpath,{libs}", "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert "magnitude 1 first 1; keys 20480 scales 1280; tile 16 waves 8 workgroups 256" in out
    assert out.count("invalid_argument:") == 4
