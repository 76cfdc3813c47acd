"""The Python binding of rope, cache and attention refuses tensors that its views would misread, before the library is
called: checked on stand-ins for device tensors, which are never looked into."""
import pytest

import splash_q4 as sq

torch = pytest.importorskip("torch")


class Device:
    """A device tensor's outside: `like` says its shape, strides and type."""

    is_cuda = True

    def __init__(self, like, at=1 << 20, device=0):
        self.like, self.at, self.device = like, at, device
        self.dtype, self.shape = like.dtype, like.shape

    def data_ptr(self):
        return self.at

    def get_device(self):
        return self.device

    def __getattr__(self, name):
        return getattr(self.like, name)


def device(*shape, dtype=torch.int32):
    return Device(torch.empty(shape, dtype=dtype))


ROW = torch.bfloat16
STORED = {sq.KV_BF16: (torch.bfloat16, torch.int16), sq.KV_INT8: (torch.int8,), sq.KV_E4M3: (torch.float8_e4m3fn, torch.int8)}


@pytest.mark.parametrize("format", STORED)
@pytest.mark.parametrize("stored", [torch.bfloat16, torch.int16, torch.float16, torch.int8, torch.float8_e4m3fn,
                                    torch.float8_e4m3fnuz, torch.float8_e5m2, torch.float32, torch.int32])
def test_pools_of_another_type(format, stored):
    shape = sq.KvShape(2, 64, 16, format)
    pool, good = device(4, 2, 16, 64, dtype=stored), device(4, 2, 16, 64, dtype=STORED[format][0])
    scales = [device(4, 2, 16, dtype=torch.float32) for _ in range(2)]
    fits = stored in STORED[format]
    for keys, values in ((pool, good), (good, pool)):
        if fits:
            assert sq.kv_cache(shape, 4, keys, values, *scales).keys.bytes == 4 * 2 * 16 * 64 * stored.itemsize
        else:
            with pytest.raises(ValueError, match="keys|values"):
                sq.kv_cache(shape, 4, keys, values, *scales)


@pytest.mark.parametrize("format", STORED)
def test_buffers_as_bytes(format):
    """What kv_cache_size counts, allocated as that many bytes."""
    shape = sq.KvShape(2, 64, 16, format)
    size = sq.kv_cache_size(shape, 4)
    buffers = [device(n, dtype=torch.uint8) for n in (size.keys, size.values, size.key_scales, size.value_scales)]
    cache = sq.kv_cache(shape, 4, *buffers)
    assert [getattr(cache, n).bytes for n in ("keys", "value_scales")] == [size.keys, size.value_scales]


@pytest.mark.parametrize("wrong", [torch.float64, torch.bfloat16, torch.int32])
def test_scales_of_another_type(wrong):
    shape, pool = sq.KvShape(2, 64, 16, sq.KV_INT8), device(4, 2, 16, 64, dtype=torch.int8)
    good, bad = device(4, 2, 16, dtype=torch.float32), device(4, 2, 16, dtype=wrong)
    sq.kv_cache(shape, 4, pool, pool, good, good)
    for scales in ((bad, good), (good, bad)):
        with pytest.raises(ValueError, match="scales"):
            sq.kv_cache(shape, 4, pool, pool, *scales)


def test_an_unknown_format():
    with pytest.raises(ValueError, match="format"):
        sq.kv_cache(sq.KvShape(2, 64, 16, 3), 4, device(8, dtype=torch.int8), device(8, dtype=torch.int8))


@pytest.mark.parametrize("wrong", [torch.float32, torch.int64, torch.bool, torch.int16])
def test_batches_of_another_type(wrong):
    starts, lengths, table = device(3), device(2), device(2, 5)
    batch = sq.kv_batch(starts, lengths, table, 4)
    assert (batch.sequences, batch.rows, batch.pages_per_sequence) == (2, 4, 5)
    sq.kv_batch(device(3, dtype=torch.uint32), lengths, table, 4)
    for at, name in enumerate(("row starts", "lengths", "page table")):
        parts = [starts, lengths, table]
        parts[at] = device(*parts[at].shape, dtype=wrong)
        with pytest.raises(ValueError, match=name):
            sq.kv_batch(*parts, 4)


def test_batches_of_other_dimensions():
    starts, lengths, table = device(3), device(2), device(2, 5)
    for parts, name in (((device(1, 3), lengths, table), "row starts"), ((starts, device(1, 2), table), "lengths"),
                        ((starts, lengths, device(10)), "page table"), ((starts, lengths, device(1, 2, 5)), "page table")):
        with pytest.raises(ValueError, match=name):
            sq.kv_batch(*parts, 4)


class Rope:
    struct = sq.Rope(64, sq.ROPE_HALF, 1.0, sq.Buffer(1 << 20, 256))


@pytest.mark.parametrize("wrong", [torch.float32, torch.int64])
def test_positions_of_another_type(wrong):
    x = device(3, 128, dtype=ROW)
    with pytest.raises(ValueError, match="positions"):
        sq.rope_add(Rope, device(3, dtype=wrong), x, x, 64, stream=0)


@pytest.mark.parametrize("raw", [True, False])
def test_the_current_stream_with_and_without_its_raw_handle(monkeypatch, raw):
    class Stream:
        cuda_stream = 0x5000

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream)
    if raw:
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0x4000 + device, raising=False)
    else:
        monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    assert sq.stream_handle().value == (0x4003 if raw else 0x5000)


def test_tensors_of_another_device(monkeypatch):
    """Without a stream of its own a call goes to the current device: tensors of another are refused, whichever they are.
    With one they are taken (and no rows mean no launch)."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(sq, "_stream_of", lambda device: 0)
    shape = sq.KvShape(2, 64, 16, sq.KV_BF16)
    pool = device(4, 2, 16, 64, dtype=ROW)
    cache, batch = sq.kv_cache(shape, 4, pool, pool), sq.kv_batch(device(3), device(2), device(2, 5), 0)
    plan = sq.attention_plan(sq.AttentionShape(2, shape, 1, 0, 0.125), 2, 3, 1)

    class Scratch:
        partials = device(plan.partials, dtype=torch.uint8)

    class FarScratch:
        partials = Device(Scratch.partials.like, device=1)

    here, far = (Device(torch.empty(3, 128, dtype=ROW), device=n) for n in (0, 1))
    words = device(3)
    calls = [lambda x, y, **kw: sq.kv_write(cache, batch, x, y, **kw),
             lambda x, y, **kw: sq.kv_read(cache, batch, x, y, **kw),
             lambda x, y, **kw: sq.kv_write(cache, batch, here, here, rope=Rope, queries=x, rotated=y, **kw),
             lambda x, y, **kw: sq.attention_add(plan, cache, batch, x, y, Scratch, **kw)]
    for run in calls:
        run(here, here)                       # no rows: checked, and nothing launched
        run(far, far, stream=0)
        for x, y in ((far, here), (here, far)):
            with pytest.raises(ValueError, match="another device"):
                run(x, y)
    for x, y, p in ((far, here, words), (here, far, words), (here, here, Device(words.like, device=1))):
        with pytest.raises(ValueError, match="another device"):
            sq.rope_add(Rope, p, x, y, 64)
    with pytest.raises(ValueError, match="another device"):
        sq.attention_add(plan, cache, batch, here, here, FarScratch)
