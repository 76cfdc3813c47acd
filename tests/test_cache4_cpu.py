"""The 4-bit cache on the host: sizes, refusals, plans, and the tensors that the Python binding takes for it."""
import ctypes

import pytest

import splash_q4 as sq
from test_attention_binding import device

torch = pytest.importorskip("torch")


def shape(**kw):
    return sq.KvShape(**{**dict(kv_heads=2, head_dim=64, page_rows=32, format=sq.KV_E2M1), **kw})


@pytest.mark.parametrize("dim,scales", [(32, 2), (64, 2), (96, 4), (128, 4), (160, 8), (192, 8), (256, 8)])
def test_sizes(dim, scales):
    size = sq.kv_cache_size(shape(head_dim=dim), 10)
    rows = 10 * 2 * 32
    assert (size.keys, size.values) == (rows * dim // 2,) * 2
    assert (size.key_scales, size.value_scales) == (rows * scales,) * 2


@pytest.mark.parametrize("dim", [16, 48, 80, 144, 240])
def test_heads_of_half_groups_are_refused(dim):
    with pytest.raises(sq.InvalidArgument, match="multiple of 32"):
        sq.kv_cache_size(shape(head_dim=dim), 4)
    with pytest.raises(sq.InvalidArgument, match="multiple of 32"):
        sq.attention_plan(sq.AttentionShape(4, shape(head_dim=dim), 1, 0, 0.1), 1, 1, 1)


@pytest.mark.parametrize("format", [3, 5, 255])
def test_other_formats_stay_unknown(format):
    with pytest.raises(sq.InvalidArgument, match="format"):
        sq.kv_cache_size(shape(format=format), 4)


@pytest.mark.parametrize("name", ["keys", "values", "key_scales", "value_scales"])
def test_short_buffers(name):
    s = shape()
    size = sq.kv_cache_size(s, 10)
    names = ("keys", "values", "key_scales", "value_scales")
    cache = sq.KvCache(s, 10, *(sq.Buffer(1 << 20, getattr(size, n) - (n == name)) for n in names))
    batch = sq.KvBatch(1, 1, 4, *(sq.Buffer(1 << 20, n) for n in (8, 4, 16)))
    rows = sq.HeadRows(sq.Buffer(1 << 20, 256), 2, 128)
    by = ctypes.byref
    with pytest.raises(sq.InvalidArgument, match=name.replace("_", " ")):
        sq.call("sq_kv_add_write", None, by(cache), by(batch), by(rows), by(rows), None, None, None)


@pytest.mark.parametrize("heads,chunk,tile", [(4, 1, 16), (32, 1, 16), (64, 1, 32), (4, 100, 128)])
def test_plans(heads, chunk, tile):
    plan = sq.attention_plan(sq.AttentionShape(heads, shape(), 1, 0, 0.125), 4, 400, chunk)
    assert plan.tile_rows == tile and plan.workgroups % 8 == 0


def test_tensors_of_the_binding():
    size = sq.kv_cache_size(shape(), 4)
    codes = [device(4, 2, 32, 32, dtype=t) for t in (torch.uint8, torch.int8, torch.float4_e2m1fn_x2)]
    scales = [device(4, 2, 32, 2, dtype=t) for t in (torch.uint8, torch.float8_e8m0fnu)]
    for c in codes:
        for s in scales:
            cache = sq.kv_cache(shape(), 4, c, c, s, s)
            assert (cache.keys.bytes, cache.value_scales.bytes) == (size.keys, size.value_scales)
    for bad in (torch.bfloat16, torch.float8_e4m3fn, torch.float32):
        with pytest.raises(ValueError, match="keys"):
            sq.kv_cache(shape(), 4, device(4, 2, 32, 32, dtype=bad), codes[0], scales[0], scales[0])
    for bad in (torch.float32, torch.bfloat16, torch.int32):
        with pytest.raises(ValueError, match="scales"):
            sq.kv_cache(shape(), 4, codes[0], codes[0], device(4, 2, 32, 2, dtype=bad), scales[0])
