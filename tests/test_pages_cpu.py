"""The pages of a cache and scored attention on the host: workspaces, and every refusal of the entry points and of the Python
binding, before anything is launched (the views point nowhere)."""
import ctypes
import math

import pytest

import splash_q4 as sq
from test_attention_binding import device
from test_attention_cpu import attention_plan, attention_shape, batch, buffer, cache, refused, rows_of

torch = pytest.importorskip("torch")
by = ctypes.byref


def pool(cache=None, sequences=3, per=4, **kw):
    c = cache if cache is not None else globals()["cache"]()
    d = dict(references=buffer(4 * c.pages), page_table=buffer(4 * sequences * per), lengths=buffer(4 * sequences),
             report=buffer(16))
    d.update(kw)
    return sq.KvPool(c, sequences, per, d["references"], d["page_table"], d["lengths"], d["report"])


def workspace_of(p):
    size = ctypes.c_uint64()
    sq.call("sq_kv_pool_workspace", by(p), by(size))
    return size.value


def test_workspace_grows_with_the_pages():
    a, b = workspace_of(pool()), workspace_of(pool(cache=cache(pages=5000)))
    assert 0 < a < b and b - a >= 3 * 4 * 4990


POOLS = [
    ("cache keys", dict(cache=dict(short="keys")), {}), ("16-byte", dict(cache=dict(at="values")), {}),
    ("sequences", dict(sequences=0), {}), ("2\\^20 sequences", dict(sequences=(1 << 20) + 1), {}),
    ("entries", dict(per=0), {}), ("2\\^28", dict(sequences=1 << 20, per=257), {}),
    ("references", {}, dict(references=buffer(39))), ("page table", {}, dict(page_table=buffer(47))),
    ("lengths", {}, dict(lengths=buffer(11))), ("report", {}, dict(report=buffer(15))),
    ("4-byte", {}, dict(references=buffer(40, (1 << 20) + 2))), ("4-byte", {}, dict(report=buffer(16, (1 << 20) + 1))),
    ("lengths", {}, dict(lengths=sq.Buffer(None, 64))),
]


@pytest.mark.parametrize("message,sizes,views", POOLS)
def test_pool_refusals(message, sizes, views):
    sizes = dict(sizes)
    if "cache" in sizes:
        sizes["cache"] = cache(**sizes["cache"])
    p, words, work = pool(**sizes, **views), buffer(8), buffer(1 << 30)
    refused("sq_kv_pool_add_release", message, by(p), words, words, 2)
    refused("sq_kv_pool_add_grow", message, by(p), words, words, 2, work)
    refused("sq_kv_pool_add_fork", message, by(p), words, words, 2, work)
    refused("sq_kv_pool_add_compact", message, by(p), work)
    with pytest.raises(sq.InvalidArgument, match=message):
        workspace_of(p)


@pytest.mark.parametrize("page_rows,per,fits", [(1024, 1 << 20, True), (1024, (1 << 20) + 1, False), (1024, 1 << 23, False),
                                                (1024, 1 << 28, False), (16, 1 << 26, True), (16, (1 << 26) + 1, False)])
def test_keys_of_a_sequence(page_rows, per, fits):
    """A pool's sequences have at most the keys of a batch's, 2^30: with more a length could grow past its 32 bits."""
    p, words = pool(cache=cache(page_rows=page_rows), sequences=1, per=per, page_table=buffer(4 * per)), buffer(8)
    if fits:
        assert workspace_of(p)
        return
    for name, rest in (("release", (words, words, 2)), ("grow", (words, words, 2, buffer(1 << 30))),
                       ("fork", (words, words, 2, buffer(1 << 30))), ("compact", (buffer(1 << 30),))):
        refused(f"sq_kv_pool_add_{name}", "2\\^30 keys", by(p), *rest)
    with pytest.raises(sq.InvalidArgument, match="2\\^30 keys"):
        workspace_of(p)


def test_request_refusals():
    p, words = pool(), buffer(8)
    size = workspace_of(p)
    work = buffer(size)
    for name, first, second in (("release", "rows to release", "keys to keep"), ("grow", "rows to grow", "keys to grow by"),
                                ("fork", "parents", "children")):
        tail = () if name == "release" else (work,)
        call = f"sq_kv_pool_add_{name}"
        refused(call, first, by(p), buffer(7), words, 2, *tail)
        refused(call, second, by(p), words, buffer(7), 2, *tail)
        refused(call, "4-byte", by(p), words, buffer(8, (1 << 20) + 2), 2, *tail)
        refused(call, "1024 requests", by(p), buffer(1 << 20), buffer(1 << 20), 1025, *tail)
        refused(call, "pool is null", None, words, words, 2, *tail)
        sq.call(call, None, by(p), sq.Buffer(None, 0), sq.Buffer(None, 0), 0, *tail) if name == "release" else None
        if tail:
            refused(call, "workspace", by(p), words, words, 2, buffer(size - 1))
            refused(call, "16-byte", by(p), words, words, 2, buffer(size, (1 << 20) + 4))
    refused("sq_kv_pool_add_compact", "workspace", by(p), buffer(size - 1))
    refused("sq_kv_pool_workspace".replace("workspace", "add_compact"), "16-byte", by(p), buffer(size, (1 << 20) + 8))


def test_calls_of_no_requests():
    """Checked like all others, and nothing is launched (the views point nowhere)."""
    p, none = pool(), sq.Buffer(None, 0)
    work = buffer(workspace_of(p))
    sq.call("sq_kv_pool_add_release", None, by(p), none, none, 0)
    for call in ("sq_kv_pool_add_grow", "sq_kv_pool_add_fork"):
        sq.call(call, None, by(p), none, none, 0, work)
        refused(call, "workspace", by(p), none, none, 0, none)
        refused(call, "lengths", by(pool(lengths=none)), none, none, 0, work)


def test_copy_refusals():
    a, pairs = cache(), buffer(16)
    refused("sq_kv_add_copy", "one shape", by(a), by(cache(page_rows=64)), pairs, 2)
    refused("sq_kv_add_copy", "one shape", by(a), by(cache(format=sq.KV_E4M3)), pairs, 2)
    refused("sq_kv_add_copy", "page pairs", by(a), by(a), buffer(15), 2)
    refused("sq_kv_add_copy", "8-byte", by(a), by(a), buffer(16, (1 << 20) + 4), 2)
    refused("sq_kv_add_copy", "key scales", by(cache(short="key_scales")), by(a), pairs, 2)
    refused("sq_kv_add_copy", "cache values", by(a), by(cache(short="values")), pairs, 2)
    refused("sq_kv_add_copy", "2\\^28", by(a), by(a), buffer(1 << 40), (1 << 28) + 1)
    refused("sq_kv_add_copy", "null", by(a), None, pairs, 2)
    sq.call("sq_kv_add_copy", None, by(a), by(a), sq.Buffer(None, 0), 0)


SCORES = [
    ("cap", dict(cap=-1.0)), ("cap", dict(cap=math.inf)), ("cap", dict(cap=math.nan)), ("cap", dict(cap=1e-38)),
    ("cap", dict(cap=3e38)), ("slopes", dict(slopes=buffer(15))), ("4-byte", dict(slopes=buffer(16, (1 << 20) + 2))),
    ("begins", dict(begins=buffer(11))), ("4-byte", dict(begins=buffer(12, (1 << 20) + 1))),
    ("prefixes", dict(prefixes=buffer(11))), ("4-byte", dict(prefixes=buffer(12, (1 << 20) + 3))),
]


@pytest.mark.parametrize("message,what", SCORES)
def test_score_refusals(message, what):
    plan, q = attention_plan(), rows_of(5, 4, 64)
    none = sq.Buffer(None, 0)
    scores = sq.AttentionScores(*[{**dict(cap=0.0, slopes=none, begins=none, prefixes=none), **what}[n]
                                  for n in ("cap", "slopes", "begins", "prefixes")])
    buffers = sq.AttentionBuffers(q, q, buffer(plan.partials))
    refused("sq_attention_add_scored", message, by(buffers), by(cache()), by(batch()), by(plan), by(scores))


def test_scored_refusals_of_the_plain_call():
    q, none = rows_of(5, 4, 64), sq.Buffer(None, 0)
    scores = sq.AttentionScores(10.0, none, none, buffer(12))
    plan = attention_plan(attention_shape(causal=0))
    buffers = sq.AttentionBuffers(q, q, buffer(plan.partials))
    refused("sq_attention_add_scored", "causal", by(buffers), by(cache()), by(batch()), by(plan), by(scores))
    plan = attention_plan()
    refused("sq_attention_add_scored", "another cache", by(buffers), by(cache(page_rows=64)), by(batch()), by(plan), by(scores))
    refused("sq_attention_add_scored", "null", None, by(cache()), by(batch()), by(plan), by(scores))
    # A scale whose quotient by the cap overflows.
    plan = attention_plan(attention_shape(scale=1e38))
    buffers = sq.AttentionBuffers(q, q, buffer(plan.partials))
    refused("sq_attention_add_scored", "cap", by(buffers), by(cache()), by(batch()), by(plan),
            by(sq.AttentionScores(0.01, none, none, none)))
    # No rows: nothing to launch.
    plan = attention_plan()
    buffers = sq.AttentionBuffers(q, q, buffer(plan.partials))
    sq.call("sq_attention_add_scored", None, by(buffers), by(cache()), by(batch(rows=0)), by(plan), by(scores))


def test_tensors_of_the_binding():
    words, good = lambda *s: device(*s), device(10)
    c = cache()
    p = sq.kv_pool(c, good, words(3, 4), words(3), words(4))
    assert (p.sequences, p.pages_per_sequence, p.page_table.bytes) == (3, 4, 48)
    for bad in ((device(10, dtype=torch.int64), words(3, 4), words(3), words(4)), (good, words(12), words(3), words(4)),
                (good, words(3, 4), words(2), words(4)), (good, words(3, 4), words(3), device(4, dtype=torch.float32)),
                (good, device(4, 3).t(), words(3), words(4)) if hasattr(torch.Tensor, "t") else ()):
        with pytest.raises((ValueError, AttributeError)):
            sq.kv_pool(c, *bad)
    with pytest.raises(ValueError, match="one length"):
        sq.kv_release(p, words(3), words(2))
    with pytest.raises(ValueError, match="requests"):
        sq.kv_release(p, device(3, dtype=torch.int64), words(3))
    with pytest.raises(ValueError, match="pairs"):
        sq.kv_copy(c, c, words(6))
    scores = sq.attention_scores(30.0, device(8, dtype=torch.float32), words(3))
    assert (scores.cap, scores.slopes.bytes, scores.begins.bytes, scores.prefixes.ptr) == (30.0, 32, 12, None)
    for kw in (dict(slopes=device(8, dtype=torch.bfloat16)), dict(begins=device(3, dtype=torch.int64)),
               dict(prefixes=device(3, 1)), dict(slopes=device(2, 4, dtype=torch.float32))):
        with pytest.raises(ValueError):
            sq.attention_scores(**kw)


def test_cxx_face(tmp_path):
    """The C++ header's pool and scores compile against the library; refusals are exceptions."""
    import pathlib
    import shutil
    import subprocess
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    exe, libs = tmp_path / "pages_check", sq.LIBRARY.parent
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(sq.HEADER.parent),
                    str(pathlib.Path(__file__).parent / "cxx_pages_check.cpp"), "-L", str(libs), "-lsplash_q4",
                    f"-Wl,-rpath,{libs}", "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert "workspace" in out and out.count("invalid_argument:") == 7
