"""The pages of a cache through the C ABI against a host simulation that takes one request after the other: books and bytes are
equal after every call, over random histories, at the edges of pages, tables and pools, with requests that cannot be carried
out, with books that contradict themselves, in graphs, and under the attention that reads the pages."""
import math

import numpy as np
import pytest

import splash_q4 as sq
from attention_oracle import bf16, from_bf16, to_bf16, torch
from pages_oracle import FORMATS, HOLE, DevicePool, Pool

pytestmark = pytest.mark.gpu


def start(seed=0, pages=60, sequences=8, per=10, **kw):
    pool = Pool(np.random.default_rng(seed), pages, sequences, per, **kw)
    return pool, DevicePool(pool)


def both(pool, device, call, *args):
    getattr(pool, call)(*args)
    getattr(device, call)(*args)
    device.check(f"{call} {args}")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kv_heads,dim,page", [(1, 32, 16), (3, 64, 32), (2, 96, 64), (2, 256, 128)])
def test_histories(fmt, kv_heads, dim, page):
    """Grow, fork, release and compact in turn, at random, in a pool that runs out of pages now and then."""
    rng = np.random.default_rng(dim + page)
    pool, device = start(page, 40, 9, 9, kv_heads=kv_heads, dim=dim, page=page, fmt=fmt)
    for step in range(60):
        n = int(rng.integers(1, 6))
        rows = rng.permutation(9)[:n]
        if rng.random() < 0.2:
            rows[-1] = rng.choice([rows[0], 9, 1 << 31])
        what = rng.choice(["grow", "grow", "fork", "release", "compact"])
        if what == "grow":
            both(pool, device, "grow", rows, rng.choice([0, 1, page - 1, page, 3 * page + 1, 20 * page], n, p=[.1, .3, .2, .2, .15, .05]))
        elif what == "fork":
            parents = rng.integers(0, 9, n)
            gone = [r for r in rows if r < 9 and r not in parents]
            if gone:        # what a child named before is released first, as a program does
                both(pool, device, "release", gone, [0] * len(gone))
            both(pool, device, "fork", parents, rows)
        elif what == "release":
            both(pool, device, "release", rows, rng.choice([0, 1, page, 2 * page + 3, 1000], n))
        else:
            both(pool, device, "compact")
        pool.check_books()


def grown(lengths, **kw):
    pool, device = start(**kw)
    both(pool, device, "grow", list(range(len(lengths))), lengths)
    return pool, device


@pytest.mark.parametrize("fmt", FORMATS)
def test_forks_share_whole_pages_and_copy_the_last(fmt):
    pool, device = grown([70, 64, 5, 0, 160], fmt=fmt)
    both(pool, device, "fork", [0, 0, 1, 2], [5, 6, 7, 3])
    assert pool.report[1] == 3 and pool.references[pool.table[0, 0]] == 3     # a full last page is shared
    assert pool.table[7, 4] == HOLE
    both(pool, device, "grow", [0, 5, 6, 3], [1, 1, 30, 2])
    both(pool, device, "release", [0], [0])
    both(pool, device, "compact")


def test_requests_that_are_not_carried_out():
    pool, device = grown([70, 64, 5, 0, 160], pages=20)          # 5 + 4 + 1 + 10 pages: none left
    assert not pool.free()
    both(pool, device, "grow", [2, 3, 2, 8, HOLE, 3], [3, 0, 1, 1, 1, 1])        # within a page; nothing; twice; nowhere; twice
    assert pool.report[0] == 4 and pool.lengths[2] == 8
    both(pool, device, "fork", [0, 1, 3, 9, 0], [5, 6, 7, 5, 3])   # no page; none needed; nothing to share; a parent that is none; a parent
    assert pool.report[0] == 3 and pool.lengths[6] == 64 and pool.lengths[5] == 0
    both(pool, device, "release", [4, 4, 99], [60, 17, 0])         # twice: the shorter
    assert pool.lengths[4] == 17 and len(pool.free()) == 8
    both(pool, device, "grow", [2, 1, 0, 3], [9 * 16, 100, 16, 1])         # eight pages: the first one's nine do not fit, nor do others
    both(pool, device, "fork", [0, 1], [0, 1])                     # itself
    assert pool.report[0] == 2
    both(pool, device, "grow", [1], [160])                         # past its row of the table
    assert pool.report[0] == 1


def test_a_shared_last_page_is_copied_before_it_grows():
    pool, device = grown([48])
    both(pool, device, "fork", [0, 0], [1, 2])
    both(pool, device, "release", [0, 1], [40, 35])                # cut inside the third page, which all three name
    both(pool, device, "grow", [0, 1, 2], [1, 20, 1])
    assert pool.report[1] == 2 and len({int(pool.table[s, 2]) for s in range(3)}) == 3
    both(pool, device, "grow", [0, 1], [0, 1])                     # their own now
    assert pool.report[1] == 0
    pool.check_books()


@pytest.mark.parametrize("pages", [1, 15, 16, 17, 4095, 4096, 4097, 16384, 40001])
def test_large_pools(pages):
    """Pools about the sizes at which the free pages are looked for and counted in several steps."""
    rng = np.random.default_rng(pages)
    pool = Pool(rng, pages, 40, max(1, pages // 8), kv_heads=1, dim=32, page=16, fmt="e2m1")
    per = pool.table.shape[1]
    order = rng.permutation(pages)
    at = 0
    for s in range(40):                                            # two thirds of the pages, anywhere
        n = min(per, pages * 2 // 3 - at, int(rng.integers(0, pages // 20 + 2)))
        pool.table[s, :n] = order[at:at + n]
        pool.references[order[at:at + n]] = 1
        pool.lengths[s] = n * 16
        at += n
    device = DevicePool(pool)
    both(pool, device, "grow", [0, 39, 7], [16, 33, 16 * (pages // 50)])
    both(pool, device, "fork", [7, 7], [20, 21])
    both(pool, device, "release", [1, 2, 3], [0, 16, 0])
    both(pool, device, "compact")
    live = int(pool.report[2])
    assert np.all(pool.references[:live]) and not np.any(pool.references[live:])
    both(pool, device, "compact")
    assert pool.report[1] == 0


def test_empty_and_full_pools():
    pool, device = start(pages=8)
    both(pool, device, "compact")
    both(pool, device, "release", [0, 1], [0, 0])
    both(pool, device, "fork", [0], [1])
    both(pool, device, "grow", [0], [128])
    both(pool, device, "compact")
    assert pool.report[2] == 8 and pool.report[1] == 0


def test_many_requests():
    """As many as a call takes, each sequence of the table among them."""
    rng = np.random.default_rng(3)
    pool = Pool(rng, 3000, 1024, 4, kv_heads=1, dim=32, page=16, fmt="e4m3")
    device = DevicePool(pool)
    both(pool, device, "grow", rng.permutation(1024), rng.integers(0, 50, 1024))
    children = rng.permutation(1024)[:500]
    both(pool, device, "release", children, [0] * 500)
    parents = np.setdiff1d(np.arange(1024), children)
    both(pool, device, "fork", rng.choice(parents, 500), children)
    both(pool, device, "compact")
    pool.check_books()
    with pytest.raises(sq.InvalidArgument, match="1024 requests"):
        device.release([0] * 1025, [0] * 1025)


def test_calls_of_no_requests():
    """They launch nothing: books, bytes and the report of the last call stay as they were."""
    pool, device = grown([70, 64, 5], pages=12)
    both(pool, device, "grow", [0, 2], [200, 1])                   # one does not fit
    report = pool.report.copy()
    assert report[0] == 1
    for call in ("release", "grow", "fork"):
        getattr(device, call)([], [])
        device.check(call)
    assert np.array_equal(device.state()["report"], report)
    graph = torch().cuda.CUDAGraph()
    words = device.words([])
    with torch().cuda.graph(graph):
        sq.kv_release(device.struct, words, words)
        sq.kv_compact(device.struct, device.scratch)
    graph.replay()
    pool.compact()
    device.check("replay")


def test_long_tables():
    """Rows of the table longer than a workgroup takes at once."""
    rng = np.random.default_rng(4)
    pool = Pool(rng, 11000, 3, 10000, kv_heads=1, dim=32, page=16, fmt="e2m1")
    device = DevicePool(pool)
    both(pool, device, "grow", [1], [16 * 9000 + 5])
    both(pool, device, "fork", [1], [2])
    both(pool, device, "release", [1], [16 * 4097 + 1])
    both(pool, device, "grow", [2, 1], [30, 5])
    both(pool, device, "compact")


@pytest.mark.parametrize("seed", range(4))
def test_books_that_contradict_themselves(seed):
    """References, entries, lengths and requests at random, whole words among them: nothing outside the views is written, and no
    call fails to end."""
    rng = np.random.default_rng(seed)
    t = torch()
    pool = Pool(rng, 50, 6, 7, kv_heads=2, dim=64, page=16, fmt="int8")
    junk = lambda *shape: rng.choice(  # noqa: E731
        np.array([0, 1, 2, 5, 6, 7, 49, 50, 111, 112, 113, 1 << 31, HOLE - 1, HOLE], np.uint32), shape).astype(np.uint32)
    pool.references, pool.table, pool.lengths = junk(50), junk(6, 7), junk(6)
    device = DevicePool(pool)
    for _ in range(8):
        device.grow(junk(9), junk(9))
        device.fork(junk(9), junk(9))
        device.release(junk(9), junk(9))
        device.compact()
        device.scratch.workspace.copy_(t.from_numpy(rng.integers(0, 256, len(device.scratch.workspace), dtype=np.uint8)))
        device.references.copy_(device.words(junk(50)))
        device.table.copy_(device.words(junk(6, 7)))
    t.cuda.synchronize()
    device.check_guards()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kv_heads,dim,page", [(1, 32, 16), (5, 96, 32), (2, 256, 256)])
def test_copy_between_caches(fmt, kv_heads, dim, page):
    rng = np.random.default_rng(dim)
    a, b = (Pool(rng, n, 1, 1, kv_heads=kv_heads, dim=dim, page=page, fmt=fmt) for n in (13, 20))
    da, db = DevicePool(a), DevicePool(b)
    pairs = np.stack([rng.integers(0, 13, 9), rng.permutation(20)[:9]], 1)
    bad = np.array([[13, 0], [0, 20], [HOLE, 1], [1, HOLE]])
    pairs = np.concatenate([pairs, bad]).astype(np.uint32)
    sq.kv_copy(da.cache, db.cache, db.words(pairs))
    for s, d in pairs:
        if s < 13 and d < 20:
            for x, y in zip(a.pools, b.pools):
                y[d] = x[s]
    da.check()
    db.check()
    sq.kv_copy(db.cache, db.cache, db.words([[int(pairs[0, 1]), int(pairs[0, 1]) ^ 1]]))    # within a cache
    for p in b.pools:
        p[int(pairs[0, 1]) ^ 1] = p[int(pairs[0, 1])]
    db.check()


def test_offsets_past_32_bits():
    """The last pages of a pool of more than 2^32 bytes."""
    t = torch()
    shape, pages = sq.KvShape(8, 128, 64, sq.KV_BF16), 40000         # 128 KiB a page of keys
    keys, values = (t.zeros((pages, 8, 64, 128), dtype=t.bfloat16, device="cuda") for _ in range(2))
    keys[pages - 2], values[pages - 2] = 3.0, 5.0
    words = lambda *s: t.zeros(s, dtype=t.int32, device="cuda")  # noqa: E731
    references, table, lengths, report = words(pages), words(2, 3), words(2), words(4)
    references[:pages - 1] = 1
    table.fill_(-1)
    table[0, 0], table[0, 1], lengths[0] = 7, pages - 2, 100
    pool = sq.kv_pool(sq.kv_cache(shape, pages, keys, values), references, table, lengths, report)
    scratch = sq.KvPoolScratch(pool)
    sq.kv_fork(pool, words(1), words(1) + 1, scratch)
    assert table[1].tolist() == [7, pages - 1, -1] and report.tolist()[:2] == [0, 1]
    assert (keys[pages - 1, :, :36] == 3).all() and (keys[pages - 1, :, 36:] == 0).all() and (values[pages - 1, :, :36] == 5).all()
    references[7:9] = 0
    table[0, 0] = table[1, 0] = 9
    sq.kv_compact(pool, scratch)
    assert report.tolist()[1:3] == [2, pages - 2] and table.tolist() == [[9, 8, -1], [9, 7, -1]]
    assert (keys[8] == 3).all() and (keys[7, :, :36] == 3).all() and (values[7, :, 36:] == 0).all()


def test_graph_replays():
    """A captured round (release, fork, grow, compact) replayed over requests that change on the device, with eager work between."""
    t = torch()
    pool, device = grown([70, 64, 5, 33, 100], pages=60)
    words = [device.words(x) for x in ([5, 6], [0, 0], [0, 1], [5, 6], [2, 5], [3, 40])]
    other = Pool(np.random.default_rng(9), 60, 8, 10)
    other.__dict__.update({k: (v.copy() if isinstance(v, np.ndarray) else [p.copy() for p in v] if isinstance(v, list) else v)
                           for k, v in pool.__dict__.items()})

    def round_():
        sq.kv_release(device.struct, words[0], words[1])
        sq.kv_fork(device.struct, words[2], words[3], device.scratch)
        sq.kv_grow(device.struct, words[4], words[5], device.scratch)
        sq.kv_compact(device.struct, device.scratch)

    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        round_()
    for parents, more in (([0, 1], [3, 40]), ([4, 4], [0, 16]), ([2, 3], [1, 1]), ([3, 0], [17, 2])):
        words[2].copy_(device.words(parents))
        words[5].copy_(device.words(more))
        graph.replay()
        pool.release([5, 6], [0, 0])
        pool.fork(parents, [5, 6])
        pool.grow([2, 5], more)
        pool.compact()
        device.check(f"replay {parents}")
        both(pool, device, "grow", [3], [1])
        both(pool, device, "release", [3], [33])


def test_on_another_stream():
    t = torch()
    pool, device = grown([70, 64, 5])
    stream = t.cuda.Stream()
    stream.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(stream):
        device.fork([0], [5])
    sq.kv_grow(device.struct, *(w := [device.words([5]), device.words([40])]), device.scratch, stream=stream.cuda_stream)
    stream.synchronize()
    pool.fork([0], [5])
    pool.grow([5], [40])
    device.check()
    del w


@pytest.mark.parametrize("fmt", FORMATS)
def test_answers_forked_from_a_prompt(fmt):
    """A prompt is written, forked three times, each fork continues with tokens of its own, one is cut back and continues, one is
    dropped, the pool is compacted: attention over every sequence is what it is over the same tokens in a cache of their own."""
    from attention_oracle import Cache, run_attention
    from cache4_oracle import Cache4
    t = torch()
    rng = np.random.default_rng(21)
    kv_heads, heads, dim, page, prompt = 2, 8, 64, 16, 75
    pool = Pool(rng, 50, 5, 12, kv_heads=kv_heads, dim=dim, page=page, fmt=fmt)
    device = DevicePool(pool)
    tokens = lambda n: bf16(rng.standard_normal((2, n, kv_heads * dim)))  # noqa: E731
    held = {0: tokens(prompt)}

    def write(s, kv):
        n = kv.shape[1]
        device.grow([s], [n])
        batch = sq.kv_batch(starts := device.words([0, n]), device.lengths[s:s + 1], device.table[s:s + 1], n)
        sq.kv_write(device.cache, batch, to_bf16(kv[0]), to_bf16(kv[1]))
        del starts

    write(0, held[0])
    device.fork([0, 0, 0], [1, 2, 4])
    for s, n in ((1, 30), (2, 5), (4, 20), (0, 1)):
        held[s] = np.concatenate([held[0][:, :prompt], new := tokens(n)], 1)
        write(s, new)
    device.release([1, 4], [80, 0])
    held[1] = np.concatenate([held[1][:, :80], new := tokens(9)], 1)
    write(1, new)
    device.compact()
    assert device.state()["report"][2] == len(np.unique(device.state()["table"][device.state()["table"] < 50]))
    q = bf16(rng.standard_normal((3, heads, dim)))
    sizes = [(1, held[s].shape[1]) for s in (0, 1, 2)]
    own = (Cache4(rng, sizes, kv_heads, dim, page) if fmt == "e2m1" else Cache(rng, sizes, kv_heads, dim, page, fmt))
    for i, s in enumerate((0, 1, 2)):
        k, v = (x.reshape(-1, kv_heads, dim).transpose(1, 0, 2) for x in held[s])
        own.k[i], own.v[i] = k, v
    want = run_attention(own.fill(), q, 1 / math.sqrt(dim))
    starts = device.words([0, 1, 2, 3])
    batch = sq.kv_batch(starts, device.lengths[:3], device.table[:3], 3)
    plan = sq.attention_plan(sq.AttentionShape(heads, pool.shape, 1, 0, 1 / math.sqrt(dim)), 3, 3, 1)
    out = t.zeros((3, heads * dim), dtype=t.bfloat16, device="cuda")
    sq.attention_add(plan, device.cache, batch, to_bf16(q.reshape(3, -1)), out, sq.AttentionScratch(plan))
    assert np.array_equal(from_bf16(out).reshape(q.shape), want)
    device.check_guards()
