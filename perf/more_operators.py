"""A serving program's paged key/value cache in 4 bits, attention with capped and biased scores over it, and the books of
its pages. Kinds of pass:

  pages      beams: sequences are dropped and others forked into their places. grow: sequences are cut back to what was
             accepted and grown again. compact: the pages in use move to the front of the pool. move: pages are copied to
             another cache.
  cache      writes the rows of new tokens into 4-bit pages and reads the same rows back in bf16; read only: a prefix
             comes back out of the cache.
  attention  the new rows' queries against the keys of their sequence: over 4-bit pages; or with scores that a tanh caps,
             that a distance lowers, keys before a sequence's first (packed documents) hidden and a prefix seen by all of
             its rows, over pages of any format.

Pages hold [kv_heads][page][dim] values. 8-bit ones stand for code * scale, one fp32 scale a token and head. 4-bit ones
hold two codes of 1, 2 and 1 bits (sign, exponent, mantissa) a byte, the first in the low half, and a byte b a group of 32
values for the scale 2^(b - 127); a row's scale bytes are 2, 4 or 8 (heads to 64, 128, 256 values).
"""
import math
import os
import sys

import torch

own = False

FORMATS = ("bf16", "int8", "e4m3", "e2m1")
LARGEST = {"int8": 127.0, "e4m3": 448.0}
HOLE = -1


# ---------------------------------------------------------------- cases

def listed():
    return [
        # A step of beam search or of sampling several answers: three kept sequences replace eight that are dropped.
        {"name": "pages_beams", "kind": "pages", "form": "beams", "fmt": "int8", "kv_heads": 8, "dim": 128, "page": 16,
         "sequences": 11, "parents": 3, "low": 400, "context": 2900, "spare": 0.2},
        # A pool whose sequences have come and gone, a third of its pages free between the others.
        {"name": "pages_compact", "kind": "pages", "form": "compact", "fmt": "bf16", "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 61, "parents": 0, "low": 300, "context": 4100, "spare": 0.33},
        # A thousand pages handed to another cache.
        {"name": "pages_move", "kind": "pages", "form": "move", "fmt": "e2m1", "kv_heads": 8, "dim": 128, "page": 64,
         "sequences": 9, "parents": 0, "low": 4000, "context": 11000, "spare": 0.1},
        # One new token of each of 32 sequences.
        {"name": "cache4_tokens", "kind": "cache", "fmt": "e2m1", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "sequences": 32, "low": 100, "context": 9000, "chunk_low": 1, "chunk": 1, "read_only": False},
        # A chunk of prompts of odd lengths.
        {"name": "cache4_prompts", "kind": "cache", "fmt": "e2m1", "heads": 40, "kv_heads": 8, "dim": 128, "page": 64,
         "sequences": 3, "low": 900, "context": 5001, "chunk_low": 301, "chunk": 1203, "read_only": False},
        # One token at the end of a long document, five query heads to a key head.
        {"name": "attend4_long", "kind": "attention", "fmt": "e2m1", "heads": 40, "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 1, "low": 131072, "context": 131072, "chunk_low": 1, "chunk": 1, "window": 0,
         "cap": 0.0, "slopes": False, "prefix": 0.0, "documents": 0},
        # One token of each of 64 conversations of ragged lengths.
        {"name": "attend4_batch", "kind": "attention", "fmt": "e2m1", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 64, "low": 200, "context": 8000, "chunk_low": 1, "chunk": 1, "window": 0,
         "cap": 0.0, "slopes": False, "prefix": 0.0, "documents": 0},
        # A full chunk at the end of a long prompt: the largest case.
        {"name": "attend4_chunk", "kind": "attention", "fmt": "e2m1", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 1, "low": 16384, "context": 16384, "chunk_low": 2048, "chunk": 2048, "window": 0,
         "cap": 0.0, "slopes": False, "prefix": 0.0, "documents": 0},
        # One token of one conversation with capped scores: the smallest attention.
        {"name": "scores_token", "kind": "attention", "fmt": "bf16", "heads": 16, "kv_heads": 8, "dim": 256,
         "page": 16, "sequences": 1, "low": 700, "context": 700, "chunk_low": 1, "chunk": 1, "window": 0,
         "cap": 50.0, "slopes": False, "prefix": 0.0, "documents": 0},
        # One token of each of 48 conversations, scores lowered by the distance, 8-bit cache.
        {"name": "scores_batch", "kind": "attention", "fmt": "int8", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 48, "low": 150, "context": 9000, "chunk_low": 1, "chunk": 1, "window": 0,
         "cap": 0.0, "slopes": True, "prefix": 0.0, "documents": 0},
        # A chunk of packed documents of odd lengths, each for itself, scores lowered by the distance.
        {"name": "scores_documents", "kind": "attention", "fmt": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 1, "low": 5003, "context": 5003, "chunk_low": 2001, "chunk": 2001, "window": 0,
         "cap": 0.0, "slopes": True, "prefix": 0.0, "documents": 11},
        # A full chunk with capped scores at the end of a long prompt, most of it a prefix that every row sees, wide heads.
        {"name": "scores_chunk", "kind": "attention", "fmt": "bf16", "heads": 16, "kv_heads": 8, "dim": 256,
         "page": 64, "sequences": 1, "low": 16384, "context": 16384, "chunk_low": 2048, "chunk": 2048, "window": 0,
         "cap": 50.0, "slopes": False, "prefix": 0.9, "documents": 0},
    ]


def draw(rng):
    def spread(lo, hi):
        """lo..hi, spread over the logarithm."""
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["pages", "pages", "cache", "attend4", "attend4", "scores", "scores", "scores"])
    fmt = "e2m1" if kind in ("cache", "attend4") else rng.choice(FORMATS)
    dims = [64, 96, 128, 128, 256] if fmt == "e2m1" else [64, 80, 96, 128, 128, 256]
    case = {"kind": kind, "fmt": fmt, "kv_heads": rng.choice([1, 2, 4, 5, 8]), "dim": rng.choice(dims),
            "page": rng.choice([16, 32, 64, 128, 256])}
    if kind == "pages":
        case["form"] = rng.choice(["beams", "grow", "compact", "move"])
        case["sequences"] = spread(4, max(4, min(64, 65536 // (case["kv_heads"] * case["dim"]))))
        case["parents"] = max(1, case["sequences"] // rng.randint(2, 4))
        case["context"] = spread(200, 4000)
        case["low"] = max(100, case["context"] // rng.choice([1, 2, 20]))
        case["spare"] = rng.uniform(0.15, 0.5)
        return case
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 5, 7, 8])
    form = rng.choice(["token", "verify", "prompt"])
    case["sequences"] = spread(1, 64) if form == "token" else rng.randint(1, 4) if form == "verify" else spread(1, 6)
    most = 100000 if form == "token" and case["sequences"] < 4 else 8000
    if form == "prompt":
        most = min(most, 8000 * 8192 // (case["heads"] * case["dim"]))
    case["context"] = spread(100, most)
    case["low"] = max(10, case["context"] // rng.choice([1, 2, 20]))
    if form == "prompt":
        most = min(case["low"], 2048 // case["sequences"])
        case["chunk"] = spread(9, most) if most > 9 else most
        case["chunk_low"] = max(1, case["chunk"] // rng.choice([1, 3]))
    else:
        case["chunk"] = case["chunk_low"] = 1 if form == "token" else 8
    if kind == "cache":
        case["read_only"] = rng.random() < 0.2
        return case
    case["kind"] = "attention"
    case["window"] = rng.choice([0, 0, 0, spread(16, 4096)])
    case.update({"cap": 0.0, "slopes": False, "prefix": 0.0, "documents": 0})
    if kind == "scores":
        what = rng.choice(["cap", "cap", "slopes", "slopes", "both", "masks"])
        if what in ("cap", "both"):
            case["cap"] = rng.choice([15.0, 30.0, 50.0])
        case["slopes"] = what in ("slopes", "both")
        if form == "prompt" and (what == "masks" or rng.random() < 0.4):
            if rng.random() < 0.5:
                case["documents"] = rng.randint(2, 16)
            else:
                case["prefix"] = rng.uniform(0.2, 1.0)
    return case


def between(lo, hi, i):
    """The i-th of the lengths spread over lo..hi (its logarithm), hi first."""
    return int(round(hi * (lo / hi) ** ((i * 0.6180339887) % 1.0)))


def lengths(case):
    """(rows, keys, first key, prefix, stored sequence) of each sequence of the batch: its new rows, and its keys with
    them. Packed documents are sequences of a batch that share a stored one."""
    out = []
    for i in range(case["sequences"]):
        keys = between(case["low"], case["context"], i)
        rows = min(keys, between(case["chunk_low"], case["chunk"], i))
        documents = case.get("documents", 0)
        if not documents:
            out.append((rows, keys, 0, int(round(case.get("prefix", 0.0) * keys)), i))
            continue
        # The documents' ends: ragged shares of the keys.
        shares = [1.0 + (j * 0.6180339887) % 1.0 * 3 for j in range(documents)]
        ends = [int(round(keys * sum(shares[:j + 1]) / sum(shares))) for j in range(documents)]
        begin = 0
        for end in ends:
            new = end - max(begin, keys - rows)
            if new > 0:
                out.append((new, end, begin, 0, i))
            begin = end
    return out


def seen(case, rows, keys, begin, prefix):
    """(pairs of rows and the keys they see, keys that any of the rows sees) of a sequence."""
    window = case["window"] or keys
    pairs, low, high = 0, keys, 0
    for p in range(keys - rows, keys):
        first, last = max(begin, p - window + 1), max(p + 1, min(prefix, keys))
        pairs += last - first
        low, high = min(low, first), max(high, last)
    return pairs, high - low


def row_bytes(case):
    """The bytes of a token's key head (or value head) in the cache."""
    dim = case["dim"]
    return {"bf16": 2 * dim, "int8": dim + 4, "e4m3": dim + 4, "e2m1": dim // 2 + dim // 32}[case["fmt"]]


def work(case):
    width = row_bytes(case)
    if case["kind"] == "pages":
        return work_of_pages(case, 2 * case["kv_heads"] * width)
    sizes = lengths(case)
    rows = sum(s[0] for s in sizes)
    if case["kind"] == "cache":
        values = 2 * rows * case["kv_heads"]
        cached, plain = values * width, values * case["dim"] * 2
        return {"bytes": cached + plain if case["read_only"] else 2 * cached + 2 * plain,
                "flops": 2 * values * case["dim"]}
    each = [seen(case, *s[:4]) for s in sizes]
    return {"bytes": 4 * rows * case["heads"] * case["dim"] + 2 * sum(k for _, k in each) * case["kv_heads"] * width,
            "flops": 4 * sum(p for p, _ in each) * case["heads"] * case["dim"]}


# ---------------------------------------------------------------- inputs

def normal(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def scale_bytes(dim):
    """The scale bytes of a 4-bit head row."""
    return 2 if dim <= 64 else 4 if dim <= 128 else 8


def groups_of(x):
    """x [..., dim] as [..., dim / 32, 32]."""
    return x.reshape(*x.shape[:-1], -1, 32)


def quantised4(x):
    """(bytes of two codes [..., dim / 2], scale bytes [..., 2, 4 or 8]) of head rows [..., dim]: the scale is the
    smallest power of two under which the largest of 32 values is at most 7 (6 is the largest code)."""
    g = groups_of(x)
    m, e = torch.frexp(g.abs().amax(-1))
    e = (e - 3 + (m > 0.875).to(e.dtype)).clamp(-125, 125)
    q = torch.ldexp(g, -e[..., None])
    size = q.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = (torch.round(size / step) * step).clamp(max=6.0)
    code = torch.where(size < 2, 2 * size, torch.where(size < 4, size + 2, size / 2 + 4)).to(torch.uint8)
    code = code + 8 * torch.signbit(q).to(torch.uint8)
    code = code.reshape(x.shape)
    scales = torch.full((*x.shape[:-1], scale_bytes(x.shape[-1])), 2, dtype=torch.uint8, device=x.device)
    scales[..., :x.shape[-1] // 32] = (e + 127).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def values4(packed, scales, dtype=torch.float32):
    """What bytes of codes [..., dim / 2] and scale bytes [..., 2, 4 or 8] stand for."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype,
                        device=packed.device)
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    g = groups_of(grid[codes.long()])
    return torch.ldexp(g, (scales[..., :g.shape[-2]].to(torch.int32) - 127)[..., None]).flatten(-2)


def quantised(x, fmt):
    """(values as stored, scales) of head rows [..., dim]."""
    if fmt == "bf16":
        return x.to(torch.bfloat16), None
    if fmt == "e2m1":
        return quantised4(x)
    largest = x.abs().amax(-1, keepdim=True)
    q = x * LARGEST[fmt] / torch.where(largest > 0, largest, 1.0)
    codes = q.round().to(torch.int8) if fmt == "int8" else q.to(torch.float8_e4m3fn)
    return codes, (largest / LARGEST[fmt])[..., 0].contiguous()


def pool_of(case, gen, pages, blank=False):
    """A pool's keys, values and their scales."""
    kv, dim = case["kv_heads"], case["dim"]
    d, shape = {}, (pages, kv, case["page"], dim)
    # A few channels of the keys are much larger than the others, as trained ones are.
    channels = 1 + 4 * (torch.rand(kv, 1, dim, device="cuda", generator=gen) > 0.97)
    for name, by in (("key", channels), ("value", 1)):
        x = torch.zeros(shape, device="cuda") if blank else normal(gen, *shape) * by
        d[name + "s"], d[name + "_scales"] = quantised(x, case["fmt"])
    d["channels"] = channels
    return d


def inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["kind"] == "pages":
        return inputs_of_pages(case, gen)
    sizes, page, dim, kv = lengths(case), case["page"], case["dim"], case["kv_heads"]
    rows = sum(s[0] for s in sizes)
    stored = {}
    for s in sizes:
        stored[s[4]] = max(stored.get(s[4], 0), -(-s[1] // page))
    most, pages = max(stored.values()), sum(stored.values()) + 8
    # The pages in an order that allocation and release have shuffled; table slots past a sequence's end name no page.
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    kept, at = torch.full((max(stored) + 1, most), HOLE, dtype=torch.int32, device="cuda"), 0
    for s, n in stored.items():
        kept[s, :n] = order[at:at + n]
        at += n
    whole = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = [0]
    for s in sizes:
        starts.append(starts[-1] + s[0])
    blank = case["kind"] == "cache" and not case["read_only"]   # a write's pages hold nothing yet
    d = pool_of(case, gen, pages, blank)
    d.update(sizes=sizes, rows=rows, pages=pages, table=kept[whole([s[4] for s in sizes]).long()].contiguous(),
             starts=whole(starts), lengths=whole([s[1] for s in sizes]), begins=whole([s[2] for s in sizes]),
             prefixes=whole([s[3] for s in sizes]))
    if case["kind"] == "attention":
        d["q"] = (normal(gen, rows, case["heads"] * dim) * 1.5).to(torch.bfloat16)
        # The heads' slopes: a geometric series down to 2^-8, every head its own.
        n = case["heads"]
        d["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / n) for h in range(n)], device="cuda")
    elif blank:   # a fused projection's rows: query, key and value heads
        x = normal(gen, rows, case["heads"] + 2 * kv, dim)
        x[:, case["heads"]:case["heads"] + kv] *= d["channels"][:, 0]
        d["qkv"] = x.to(torch.bfloat16).reshape(rows, -1)
    return d


def prepare(case, seed):
    d = inputs(case, seed)
    state = {"case": case, "d": d}
    if not own:
        return state
    sys.path.insert(0, os.path.join(os.getcwd(), "splash-desktop_amd"))
    import splash_q4 as sq
    state["sq"] = sq
    fmt = {"bf16": sq.KV_BF16, "int8": sq.KV_INT8, "e4m3": sq.KV_E4M3, "e2m1": sq.KV_E2M1}[case["fmt"]]
    shape = sq.KvShape(kv_heads=case["kv_heads"], head_dim=case["dim"], page_rows=case["page"], format=fmt)
    state["cache"] = sq.kv_cache(shape, d["pages"], d["keys"], d["values"], d["key_scales"], d["value_scales"])
    if case["kind"] == "pages":
        if case["form"] == "move":
            t = d["to"]
            state["to"] = sq.kv_cache(shape, t["pages"], t["keys"], t["values"], t["key_scales"], t["value_scales"])
        else:
            state["pool"] = sq.kv_pool(state["cache"], d["references"], d["table"], d["lengths"], d["report"])
            state["scratch"] = sq.KvPoolScratch(state["pool"])
        return state
    empty = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    state["batch"] = sq.kv_batch(d["starts"], d["lengths"], d["table"], d["rows"])
    if case["kind"] == "cache":
        state["k"], state["v"] = (empty(d["rows"], case["kv_heads"] * case["dim"]) for _ in range(2))
        return state
    attention = sq.AttentionShape(heads=case["heads"], kv=shape, window=case["window"], causal=1,
                                  scale=1 / math.sqrt(case["dim"]))
    state["plan"] = sq.attention_plan(attention, len(d["sizes"]), d["rows"], max(s[0] for s in d["sizes"]))
    state["scratch"] = sq.AttentionScratch(state["plan"])
    state["out"] = empty(d["rows"], case["heads"] * case["dim"])
    if case["cap"] or case["slopes"] or case["prefix"] or case["documents"]:
        state["scores"] = sq.attention_scores(cap=case["cap"], slopes=d["slopes"] if case["slopes"] else None,
                                              begins=d["begins"] if case["documents"] else None,
                                              prefixes=d["prefixes"] if case["prefix"] else None)
    return state


# ---------------------------------------------------------------- passes

def run(state):
    return run_own(state) if own else run_plain(state)


def run_own(state):
    sq, case, d = state["sq"], state["case"], state["d"]
    if case["kind"] == "attention":
        sq.attention_add(state["plan"], state["cache"], state["batch"], d["q"], state["out"], state["scratch"],
                         scores=state.get("scores"))
        return state["out"]
    if case["kind"] == "cache":
        if not case["read_only"]:
            q, kv = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
            sq.kv_write(state["cache"], state["batch"], d["qkv"][:, q:q + kv], d["qkv"][:, q + kv:])
        sq.kv_read(state["cache"], state["batch"], state["k"], state["v"])
        return [state["k"], state["v"]]
    if case["form"] == "move":
        sq.kv_copy(state["cache"], state["to"], d["pairs"])
        return outputs_of_pages(d["to"])
    if case["form"] == "beams":
        sq.kv_release(state["pool"], d["children"], d["keeps"])
        sq.kv_fork(state["pool"], d["parents"], d["children"], state["scratch"])
    elif case["form"] == "grow":
        sq.kv_release(state["pool"], d["growing"], d["keeps"])
        sq.kv_grow(state["pool"], d["growing"], d["more"], state["scratch"])
    else:
        d["books"].copy_(d["fragmented"])   # every pass meets the pool as its sequences have left it
        sq.kv_compact(state["pool"], state["scratch"])
    return outputs_of_pages(d)


def places(d, case):
    """(page, row in it) of each of the batch's rows."""
    pages, rows = [], []
    for s, (n, keys, *_) in enumerate(d["sizes"]):
        p = torch.arange(keys - n, keys, device="cuda")
        pages.append(d["table"][s, p // case["page"]].long())
        rows.append(p % case["page"])
    return torch.cat(pages), torch.cat(rows)


def stored_values(d, name, fmt, pick):
    """The fp32 values that pick(tensor) of a pool's keys or values stands for."""
    t = d[name + "s"]
    if fmt == "e4m3":
        t = pick(t.view(torch.uint8)).view(t.dtype).float()
    elif fmt == "e2m1":
        return values4(pick(t), pick(d[name + "_scales"]))
    else:
        t = pick(t).float()
    return t if fmt == "bf16" else t * pick(d[name + "_scales"])[..., None]


def run_plain(state):
    case, d = state["case"], state["d"]
    if case["kind"] == "pages":
        return pages_plain(case, d)
    if case["kind"] == "attention":
        return attend_plain(case, d)
    rows, dim, kv = d["rows"], case["dim"], case["kv_heads"]
    page, slot = places(d, case)
    if not case["read_only"]:
        _, k, v = d["qkv"].float().reshape(rows, -1, dim).split([case["heads"], kv, kv], 1)
        for name, t in (("key", k), ("value", v)):
            codes, scales = quantised4(t)
            d[name + "s"][page, :, slot] = codes
            d[name + "_scales"][page, :, slot] = scales
    return [stored_values(d, name, "e2m1", lambda t: t[page, :, slot]).reshape(rows, -1).to(torch.bfloat16)
            for name in ("key", "value")]


def attend_plain(case, d):
    dim, kv, group = case["dim"], case["kv_heads"], case["heads"] // case["kv_heads"]
    out, at = [], 0
    for s, (n, keys, begin, prefix, _) in enumerate(d["sizes"]):
        pages = d["table"][s, :-(-keys // case["page"])].long()

        def cached(name):
            t = stored_values(d, name, case["fmt"], lambda t: t[pages])
            return t.transpose(0, 1).reshape(kv, -1, dim)[:, begin:keys]

        q = d["q"][at:at + n].float().reshape(n, kv, group, dim).permute(1, 2, 0, 3).reshape(kv, group * n, dim)
        scores = torch.bmm(q, cached("key").transpose(1, 2).contiguous()) * (1 / math.sqrt(dim))
        if case["cap"]:
            scores = torch.tanh(scores / case["cap"]) * case["cap"]
        scores = scores.reshape(kv, group, n, keys - begin)
        row, key = torch.arange(keys - n, keys, device="cuda")[:, None], torch.arange(begin, keys, device="cuda")
        if case["slopes"]:
            scores = scores - d["slopes"].reshape(kv, group, 1, 1) * (row - key).abs()
        hidden = (key > row) & (key >= prefix)
        if case["window"]:
            hidden = hidden | (key <= row - case["window"])
        scores = scores.masked_fill_(hidden, -math.inf)
        weights = torch.exp_(scores.sub_(scores.amax(-1, keepdim=True)))
        total = weights.sum(-1, keepdim=True)
        o = torch.bmm(weights.reshape(kv, group * n, -1), cached("value")).reshape(kv, group, n, dim) / total
        out.append(o.permute(2, 0, 1, 3).reshape(n, -1).to(torch.bfloat16))
        at += n
    return torch.cat(out)


# ---------------------------------------------------------------- the pool's pages

def inputs_of_pages(case, gen):
    """A pool with its books: how many table entries name each page, the table, the keys of each sequence, and what a call
    reports. Its free pages lie between the others."""
    page, form, n = case["page"], case["form"], case["sequences"]
    sizes = [between(case["low"], case["context"], i) for i in range(n)]
    used = [-(-k // page) for k in sizes]
    if form == "beams":     # the first sequences are kept, the others are earlier forks of them
        sizes = [sizes[i % case["parents"]] for i in range(n)]
        used = [used[i % case["parents"]] for i in range(n)]
    most, live = max(used) + 16, sum(used)
    pages = int(math.ceil(live / (1 - case["spare"]))) + 16 * n
    if form == "compact":
        pages -= 16 * n
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table, at = torch.full((n, most), HOLE, dtype=torch.int32), 0
    order_h = order.cpu()
    for s in range(n):
        parent = s % case["parents"] if form == "beams" else s
        shared = sizes[parent] // page if parent != s else 0
        table[s, :shared] = table[parent, :shared]
        table[s, shared:used[s]] = order_h[at:at + used[s] - shared]
        at += used[s] - shared
    named = table[table != HOLE].long()
    references = torch.zeros(pages, dtype=torch.int32)
    references.index_add_(0, named, torch.ones_like(named, dtype=torch.int32))
    d = pool_of(case, gen, pages)
    # The books in one tensor, its parts the views that the calls take.
    books = torch.cat([references, table.flatten(), torch.tensor(sizes, dtype=torch.int32),
                       torch.zeros(4, dtype=torch.int32)]).cuda()
    d["books"], d["fragmented"], d["pages"] = books, books.clone(), pages
    parts = books.split([pages, n * most, n, 4])
    d["references"], d["table"], d["lengths"], d["report"] = parts[0], parts[1].view(n, most), parts[2], parts[3]
    whole = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    if form == "beams":
        children = list(range(case["parents"], n))
        d["children"] = whole(children)
        d["parents"] = torch.randint(0, case["parents"], (len(children),), device="cuda", generator=gen).to(torch.int32)
        d["keeps"] = torch.zeros_like(d["children"])
    elif form == "grow":
        growing = list(range(n - case["parents"], n))
        d["growing"], d["keeps"] = whole(growing), whole([sizes[s] for s in growing])
        d["more"] = torch.randint(1, 15 * page, (len(growing),), device="cuda", generator=gen).to(torch.int32)
    elif form == "move":
        d["to"] = pool_of(case, gen, pages)
        d["to"]["pages"] = pages
        moved = order[:live].to(torch.int32)
        d["pairs"] = torch.stack([moved, torch.randperm(pages, device="cuda", generator=gen)[:live].to(torch.int32)],
                                 1).contiguous()
    return d


def work_of_pages(case, token):
    """What the form cannot do without; token: a token's bytes in the cache."""
    page, n = case["page"], case["sequences"]
    sizes = [between(case["low"], case["context"], i) for i in range(n)]
    used = [-(-k // page) for k in sizes]
    live = sum(used)
    if case["form"] == "beams":
        kept = [sizes[i] for i in range(case["parents"])]
        mean = sum(kept) / len(kept)
        children = n - case["parents"]
        entries = children * sum(-(-k // page) for k in kept) / len(kept)
        rest = sum(k % page for k in kept) / len(kept)
        # Entries dropped (read, written, counted down) and copied (read, written, counted up), tokens of the last pages.
        return {"bytes": int(entries * 4 * 8 + children * rest * token * 2), "flops": int(2 * entries + mean)}
    if case["form"] == "grow":
        entries = case["parents"] * 8
        return {"bytes": entries * 4 * 8 + 4 * live, "flops": 2 * entries}
    if case["form"] == "move":
        return {"bytes": 2 * live * page * token + 8 * live, "flops": live}
    moved = live * case["spare"]   # of the live pages, as many lie past the first `live` places
    return {"bytes": int(2 * moved * page * token + 4 * live / (1 - case["spare"]) + 8 * live), "flops": int(2 * live)}


def outputs_of_pages(d):
    """The pool as it is now, its bits as whole numbers (they are moved, not computed), and its books where it has some."""
    whole = {1: torch.uint8, 2: torch.int16, 4: torch.int32}
    out = [d[name].view(whole[d[name].element_size()]) for name in ("keys", "values", "key_scales", "value_scales") if d[name] is not None]
    return out + [d[name] for name in ("references", "table", "lengths", "report") if name in d]


def copy_pages(source, to, pairs, rows=None):
    """Pages pairs[:, 0] of one pool into pages pairs[:, 1] of another (or of itself); rows: the rows of each, all of them
    where there is None."""
    for name in ("keys", "values", "key_scales", "value_scales"):
        if source[name] is None:
            continue
        a, b = source[name], to[name]
        if a.dtype == torch.float8_e4m3fn:
            a, b = a.view(torch.uint8), b.view(torch.uint8)
        moved = a[pairs[:, 0].long()]
        if rows is not None:
            inside = torch.arange(a.shape[2], device="cuda")[None] < rows[:, None]          # [pairs, rows of a page]
            inside = inside[:, None, :] if a.dim() == 3 else inside[:, None, :, None]
            moved = torch.where(inside, moved, b[pairs[:, 1].long()])
        b[pairs[:, 1].long()] = moved


def drop(d, sequences, keeps, page):
    """The sequences' entries past their first `keeps` keys."""
    entry = torch.arange(d["table"].shape[1], device="cuda")[None]
    mine = d["table"][sequences.long()]
    gone = (entry >= ((keeps + page - 1) // page)[:, None]) & (mine != HOLE)
    pages = mine[gone].long()
    d["references"].index_add_(0, pages, torch.full_like(mine[gone], -1))
    d["table"][sequences.long()] = torch.where(gone, HOLE, mine)
    d["lengths"][sequences.long()] = torch.minimum(d["lengths"][sequences.long()], keeps)


def pages_plain(case, d):
    page = case["page"]
    if case["form"] == "move":
        copy_pages(d, d["to"], d["pairs"])
        return outputs_of_pages(d["to"])
    report = [0, 0, 0, 0]
    if case["form"] == "beams":
        drop(d, d["children"], d["keeps"], page)
        # Whole pages are shared, and the last one, which the child goes on writing, is copied to the lowest free pages.
        parents, children = d["parents"].long(), d["children"].long()
        keys, entry = d["lengths"][parents], torch.arange(d["table"].shape[1], device="cuda")[None]
        mine = torch.where(entry < (keys // page)[:, None], d["table"][parents], HOLE)
        shared = mine[mine != HOLE]
        free = torch.nonzero(d["references"] == 0)[:, 0].to(torch.int32)
        d["references"].index_add_(0, shared.long(), torch.ones_like(shared))
        part = torch.nonzero(keys % page)[:, 0]
        new = free[:part.numel()]
        last = (keys // page)[part].long()
        copy_pages(d, d, torch.stack([d["table"][parents[part], last], new], 1), (keys % page)[part])
        mine[part, last] = new
        d["references"][new.long()] = 1
        d["table"][children] = mine
        d["lengths"][children] = keys
        report[1] = part.numel()
    elif case["form"] == "grow":
        drop(d, d["growing"], d["keeps"], page)
        s = d["growing"].long()
        keys = d["lengths"][s]
        first, last = (keys + page - 1) // page, (keys + d["more"] + page - 1) // page
        entry = torch.arange(d["table"].shape[1], device="cuda")[None]
        wanted = (entry >= first[:, None]) & (entry < last[:, None])
        new = torch.nonzero(d["references"] == 0)[:, 0].to(torch.int32)[:int(wanted.sum())]
        mine = d["table"][s]
        mine[wanted] = new
        d["table"][s] = mine
        d["references"][new.long()] = 1
        d["lengths"][s] = keys + d["more"]
    else:
        d["books"].copy_(d["fragmented"])
        # The last page in use goes to the first free place, the one before it to the second, and so on.
        used = torch.nonzero(d["references"])[:, 0]
        free = torch.nonzero(d["references"] == 0)[:, 0]
        live = used.numel()
        to = free[free < live]
        source = used.flip(0)[:to.numel()]
        copy_pages(d, d, torch.stack([source, to], 1))
        place = torch.arange(d["pages"], device="cuda", dtype=torch.int32)
        place[source] = to.to(torch.int32)
        d["references"][to] = d["references"][source]
        d["references"][source] = 0
        named = d["table"] != HOLE
        d["table"][named] = place[d["table"][named].long()]
        report[1], report[2] = to.numel(), live
    d["report"].copy_(torch.tensor(report, dtype=torch.int32))
    return outputs_of_pages(d)


# ---------------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    if case["kind"] == "pages":
        return None     # nothing is computed: bits are moved and whole numbers counted
    d = inputs(case, seed)
    return exact_cache(case, d) if case["kind"] == "cache" else exact_attention(case, d)


GRID = sorted({s * v for s in (-1.0, 1.0) for v in (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)})


def nearest4(t):
    """[..., dim] as its groups' codes and scales stand for it: the nearest value, ties to the even code."""
    g = t.reshape(*t.shape[:-1], -1, 32)
    top = g.abs().amax(-1, keepdim=True)
    # The least whole exponent whose 7 / 8 of the next power of two above the largest code holds the largest value.
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 7.0))
    e = torch.where(torch.exp2(e - 1) * 7 >= top, e - 1, torch.where(torch.exp2(e) * 7 < top, e + 1, e))
    scale = torch.exp2(torch.where(top > 0, e, -125.0).clamp(-125.0, 125.0))
    q = g / scale
    grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")
    above = torch.searchsorted(grid, q.contiguous()).clamp(1, grid.numel() - 1)
    lo, hi = grid[above - 1], grid[above]
    # Fifteen values, zero (code 0, even) at index 7: a code's last bit is that of its distance from there.
    even = torch.where((above - 1 - 7) % 2 == 0, lo, hi)
    return (torch.where(q - lo < hi - q, lo, torch.where(q - lo > hi - q, hi, even)) * scale).reshape(t.shape)


def read4(codes, scales):
    """Bytes of codes and scales as 64-bit values, bit by bit."""
    c = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
    sign, exponent, mantissa = c // 8, c // 2 % 4, c % 2
    size = torch.where(exponent == 0, mantissa * 0.5, torch.exp2(exponent.double() - 1) * (1 + mantissa * 0.5))
    by = torch.exp2(scales.double() - 127.0).repeat_interleave(32, -1)[..., :c.shape[-1]]
    return torch.where(sign == 1, -size, size) * by


def exact_cache(case, d):
    rows, dim, kv, heads = d["rows"], case["dim"], case["kv_heads"], case["heads"]
    if case["read_only"]:
        out = []
        for values, scales in (("keys", "key_scales"), ("values", "value_scales")):
            parts = []
            for s, (n, keys, *_) in enumerate(d["sizes"]):
                for p in range((keys - n) // case["page"], -(-keys // case["page"])):
                    at = int(d["table"][s, p])
                    lo, hi = max(0, keys - n - p * case["page"]), min(case["page"], keys - p * case["page"])
                    parts.append(read4(d[values][at], d[scales][at])[:, lo:hi].transpose(0, 1))
            out.append(torch.cat(parts).flatten(1))
        return out
    x = d["qkv"].reshape(rows, heads + 2 * kv, dim)
    return [nearest4(x[:, at:at + kv].double()).flatten(1) for at in (heads, heads + kv)]


def exact_attention(case, d):
    dim, kv = case["dim"], case["kv_heads"]
    group, page = case["heads"] // kv, case["page"]
    out = torch.empty((d["rows"], case["heads"], dim), dtype=torch.float64, device="cuda")
    at = 0
    for s, (n, keys, begin, prefix, _) in enumerate(d["sizes"]):
        position = torch.arange(begin, keys, device="cuda")
        where, slot = d["table"][s].long()[position // page], position % page
        rows = torch.arange(keys - n, keys, device="cuda")[:, None]
        allowed = (position[None] <= rows) | (position[None] < prefix)
        if case["window"]:
            allowed &= position[None] > rows - case["window"]
        for h in range(kv):
            kvs = []
            for name in ("key", "value"):
                t, by = d[name + "s"], d[name + "_scales"]
                if case["fmt"] == "e2m1":
                    kvs.append(read4(t[where, h, slot], by[where, h, slot]))
                    continue
                t = t.view(torch.uint8)[where, h, slot].view(t.dtype) if case["fmt"] == "e4m3" else t[where, h, slot]
                kvs.append(t.double() if by is None else t.double() * by[where, h, slot].double()[:, None])
            k, v = kvs
            for g in range(group):
                head = h * group + g
                q = d["q"][at:at + n].reshape(n, -1, dim)[:, head].double()
                logits = (q @ k.T) / math.sqrt(dim)
                if case["cap"]:
                    logits = case["cap"] * torch.tanh(logits / case["cap"])
                if case["slopes"]:
                    logits = logits - d["slopes"][head].double() * (rows - position[None]).abs().double()
                logits[~allowed] = -math.inf
                out[at:at + n, head] = torch.softmax(logits, -1) @ v
        at += n
    return out.flatten(1)
