"""Attention over a paged key/value cache, with what comes before it: rotary positions, and the cache that is written
in 16 or 8 bits and read back. The cases are a serving program's: single tokens, verify lanes of 8 rows, prompts in
chunks of up to 2048 rows, over contexts from a few tokens to a long document's.

Three kinds of pass:
  rope       rotates a fused projection's query and key heads into another tensor.
  cache      writes the rows of new tokens into the cache's pages (rotating keys and queries on the way where the case
             has a rope) and reads the same rows back in bf16; read only: a prefix comes back out of the cache.
  attention  the new rows' queries against every key of their sequence in the cache, their own among them.

Pages hold [kv_heads][page][dim] values; 8-bit ones stand for code * scale, one fp32 scale a token and head.
"""
import math
import os
import sys

import torch

own = False

FORMATS = ("bf16", "int8", "e4m3")
LARGEST = {"int8": 127.0, "e4m3": 448.0}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # One token's query and key heads, the smallest call: latency alone.
        {"name": "rope_token", "kind": "rope", "rows": 1, "heads": 40, "dim": 128, "rotary": 128, "layout": "half",
         "scaling": "none", "base": 10000.0, "far": 4000},
        # A full chunk far into a document, half of each head rotated in interleaved pairs, scaled for long contexts.
        {"name": "rope_chunk", "kind": "rope", "rows": 2048, "heads": 40, "dim": 128, "rotary": 64,
         "layout": "interleaved", "scaling": "yarn", "base": 1000000.0, "far": 1000000},
        # One new token of each of 32 sequences into an 8-bit cache.
        {"name": "cache_tokens", "kind": "cache", "fmt": "int8", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "sequences": 32, "low": 100, "context": 9000, "chunk_low": 1, "chunk": 1, "rope": False, "read_only": False},
        # Verify lanes of eight rows, keys and queries rotated on the way into a bf16 cache.
        {"name": "cache_verify", "kind": "cache", "fmt": "bf16", "heads": 16, "kv_heads": 2, "dim": 256, "page": 64,
         "sequences": 4, "low": 300, "context": 20000, "chunk_low": 8, "chunk": 8, "rope": True, "read_only": False},
        # A chunk of prompts of odd lengths into an e4m3 cache.
        {"name": "cache_chunk", "kind": "cache", "fmt": "e4m3", "heads": 40, "kv_heads": 8, "dim": 128, "page": 64,
         "sequences": 3, "low": 900, "context": 5001, "chunk_low": 301, "chunk": 1203, "rope": False,
         "read_only": False},
        # A long prefix read back, as a program does that moves it to another cache.
        {"name": "cache_prefix", "kind": "cache", "fmt": "int8", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "sequences": 1, "low": 29999, "context": 29999, "chunk_low": 29999, "chunk": 29999, "rope": False,
         "read_only": True},
        # One token of one conversation: the smallest attention.
        {"name": "attend_token", "kind": "attention", "fmt": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "sequences": 1, "low": 700, "context": 700, "chunk_low": 1, "chunk": 1, "window": 0},
        # One token of each of 64 conversations of ragged lengths over an e4m3 cache.
        {"name": "attend_batch", "kind": "attention", "fmt": "e4m3", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 64, "low": 200, "context": 8000, "chunk_low": 1, "chunk": 1, "window": 0},
        # One token at the end of a long document, 8-bit cache, five query heads to a key head.
        {"name": "attend_long", "kind": "attention", "fmt": "int8", "heads": 40, "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 1, "low": 131072, "context": 131072, "chunk_low": 1, "chunk": 1, "window": 0},
        # Four verify lanes of eight rows, wide heads, bf16 cache.
        {"name": "attend_verify", "kind": "attention", "fmt": "bf16", "heads": 16, "kv_heads": 2, "dim": 256,
         "page": 64, "sequences": 4, "low": 1500, "context": 20000, "chunk_low": 8, "chunk": 8, "window": 0},
        # Prompts of odd lengths in one chunk, narrow heads, a sliding window, 8-bit cache.
        {"name": "attend_prompts", "kind": "attention", "fmt": "int8", "heads": 64, "kv_heads": 8, "dim": 64,
         "page": 32, "sequences": 5, "low": 37, "context": 3001, "chunk_low": 37, "chunk": 999, "window": 1024},
        # A full chunk at the end of a long prompt: the largest case.
        {"name": "attend_chunk", "kind": "attention", "fmt": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 1, "low": 16384, "context": 16384, "chunk_low": 2048, "chunk": 2048, "window": 0},
    ]


def draw(rng):
    def spread(lo, hi, step=1):
        """lo..hi, a multiple of step, spread over the logarithm."""
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return max(lo, min(hi, int(round(v / step)) * step))

    kind = rng.choice(["rope", "cache", "cache", "attention", "attention", "attention"])
    if kind == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        return {"kind": "rope", "rows": spread(1, 2048), "heads": rng.randint(1, 48), "dim": dim,
                "rotary": rng.choice([dim, dim // 2]), "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "yarn"]), "base": rng.choice([10000.0, 500000.0, 1000000.0]),
                "far": spread(100, 1000000)}
    kv_heads, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 5, 7, 8])
    case = {"kind": kind, "fmt": rng.choice(FORMATS), "heads": kv_heads * group, "kv_heads": kv_heads,
            "dim": rng.choice([64, 64, 80, 96, 128, 128, 128, 256]), "page": rng.choice([16, 32, 64, 128, 256])}
    form = rng.choice(["token", "verify", "prompt"])
    case["sequences"] = spread(1, 64) if form == "token" else rng.randint(1, 4) if form == "verify" else spread(1, 6)
    case["context"] = spread(100, 100000 if form == "token" and case["sequences"] < 4 else 8000)
    case["low"] = max(10, case["context"] // rng.choice([1, 2, 20]))
    if form == "prompt":
        most = min(case["low"], 2048 // case["sequences"])
        case["chunk"] = spread(9, most) if most > 9 else most
        case["chunk_low"] = max(1, case["chunk"] // rng.choice([1, 3]))
    else:
        case["chunk"] = case["chunk_low"] = 1 if form == "token" else 8
    if kind == "cache":
        case["rope"], case["read_only"] = case["fmt"] == "bf16" and rng.random() < 0.5, rng.random() < 0.2
        if case["read_only"]:
            case["rope"] = False
    else:
        case["window"] = rng.choice([0, 0, 0, spread(16, 4096)])
    return case


def between(lo, hi, i):
    """The i-th of the lengths spread over lo..hi (its logarithm), hi first."""
    return int(round(hi * (lo / hi) ** ((i * 0.6180339887) % 1.0)))


def lengths(case):
    """(rows, keys) of each sequence: its new rows, and its keys with them."""
    out = []
    for i in range(case["sequences"]):
        keys = between(case["low"], case["context"], i)
        out.append((min(keys, between(case["chunk_low"], case["chunk"], i)), keys))
    return out


def seen(case, rows, keys):
    """(pairs of rows and the keys they see, keys that any of the rows sees) of a sequence."""
    window = case["window"] or keys
    pairs = sum(min(window, p + 1) for p in range(keys - rows, keys))
    return pairs, keys - max(0, keys - rows - window + 1)


def work(case):
    if case["kind"] == "rope":
        values = case["rows"] * case["heads"] * case["dim"]
        rotated = case["rows"] * case["heads"] * case["rotary"]
        return {"bytes": 4 * values + 4 * case["rows"] + 4 * case["rotary"], "flops": 3 * rotated}
    width = case["dim"] * (2 if case["fmt"] == "bf16" else 1) + (0 if case["fmt"] == "bf16" else 4)
    sizes = lengths(case)
    rows = sum(r for r, _ in sizes)
    if case["kind"] == "cache":
        values = 2 * rows * case["kv_heads"]
        cached, plain = values * width, values * case["dim"] * 2
        queries = 4 * rows * case["heads"] * case["dim"] if case["rope"] else 0
        flops = rows * (case["kv_heads"] + case["heads"]) * case["dim"] * 3 if case["rope"] else 0
        return {"bytes": cached + plain if case["read_only"] else 2 * cached + 2 * plain + queries,
                "flops": flops + 2 * values * case["dim"]}
    pairs = sum(seen(case, *s)[0] for s in sizes)
    keys = sum(seen(case, *s)[1] for s in sizes)
    return {"bytes": 4 * rows * case["heads"] * case["dim"] + 2 * keys * case["kv_heads"] * width,
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---------------------------------------------------------------- inputs

def normal(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def quantised(x, fmt):
    """(values as stored, fp32 scales) of head rows [..., dim]."""
    if fmt == "bf16":
        return x.to(torch.bfloat16), None
    largest = x.abs().amax(-1, keepdim=True)
    q = x * LARGEST[fmt] / torch.where(largest > 0, largest, 1.0)
    codes = q.round().to(torch.int8) if fmt == "int8" else q.to(torch.float8_e4m3fn)
    return codes, (largest / LARGEST[fmt])[..., 0].contiguous()


def inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["kind"] == "rope":
        d = {"x": normal(gen, case["rows"], case["heads"] * case["dim"]).to(torch.bfloat16)}
        first = torch.randint(0, max(1, case["far"] - case["rows"]), (1,), device="cuda", generator=gen)
        d["positions"] = (first + torch.arange(case["rows"], device="cuda")).to(torch.int32)
        return d
    sizes, page, dim, kv = lengths(case), case["page"], case["dim"], case["kv_heads"]
    rows, most = sum(r for r, _ in sizes), max(-(-k // page) for _, k in sizes)
    needed = sum(-(-k // page) for _, k in sizes)
    pages = needed + 8
    # The pages in an order that allocation and release have shuffled; table slots past a sequence's end name no page.
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table, at = torch.full((len(sizes), most), -1, dtype=torch.int32, device="cuda"), 0
    for s, (_, keys) in enumerate(sizes):
        n = -(-keys // page)
        table[s, :n] = order[at:at + n]
        at += n
    starts = [0]
    for r, _ in sizes:
        starts.append(starts[-1] + r)
    d = {"sizes": sizes, "rows": rows, "pages": pages, "table": table,
         "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
         "lengths": torch.tensor([k for _, k in sizes], dtype=torch.int32, device="cuda")}
    # A few channels of the keys are much larger than the others, as trained ones are.
    channels = 1 + 4 * (torch.rand(kv, 1, dim, device="cuda", generator=gen) > 0.97)
    pool = (pages, kv, page, dim)
    blank = case["kind"] == "cache" and not case["read_only"]
    if blank:   # a write's pages hold what was there before: nothing yet
        stored = torch.bfloat16 if case["fmt"] == "bf16" else torch.int8 if case["fmt"] == "int8" else torch.float8_e4m3fn
        d["keys"], d["values"] = (torch.zeros(pool, device="cuda").to(stored) for _ in range(2))
        d["key_scales"], d["value_scales"] = (torch.zeros(pool[:3], device="cuda") for _ in range(2))
    else:
        d["keys"], d["key_scales"] = quantised(normal(gen, *pool) * channels, case["fmt"])
        d["values"], d["value_scales"] = quantised(normal(gen, *pool), case["fmt"])
    if case["kind"] == "attention":
        d["q"] = (normal(gen, rows, case["heads"] * dim) * 1.5).to(torch.bfloat16)
    elif blank:   # a fused projection's rows: query, key and value heads
        x = normal(gen, rows, case["heads"] + 2 * kv, dim)
        x[:, case["heads"]:case["heads"] + kv] *= channels[:, 0]
        d["qkv"] = x.to(torch.bfloat16).reshape(rows, -1)
    return d


def frequencies(case):
    """(radians a position of each pair, in 64 bits; the factor of cosine and sine) of a rope."""
    d, base, factor, original = case["rotary"], case["base"], 8.0, 32768
    f = torch.tensor([base ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "yarn":
        turning = lambda turns: d * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(turning(32.0)), 0), min(math.ceil(turning(1.0)), d - 1)
        ramp = ((torch.arange(d // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def rope_case(case):
    """The rope of a cache case that has one."""
    return {"rotary": case["dim"], "base": 1000000.0, "scaling": "none", "layout": "half"}


def prepare(case, seed):
    d = inputs(case, seed)
    state = {"case": case, "d": d}
    rope = case if case["kind"] == "rope" else rope_case(case) if case.get("rope") else None
    if not own:
        if rope:
            f, state["magnitude"] = frequencies(rope)
            state["frequencies"] = f.cuda()
        return state
    sys.path.insert(0, os.path.join(os.getcwd(), "splash-desktop_amd"))
    import splash_q4 as sq
    state["sq"] = sq
    if rope:
        layout = {"half": sq.ROPE_HALF, "interleaved": sq.ROPE_INTERLEAVED}[rope["layout"]]
        scaling = {"none": sq.ROPE_SCALING_NONE, "linear": sq.ROPE_SCALING_LINEAR, "yarn": sq.ROPE_SCALING_YARN}
        config = sq.RopeConfig(rotary_dim=rope["rotary"], layout=layout, scaling=scaling[rope["scaling"]],
                               base=rope["base"], factor=8.0, original_positions=32768)
        state["rope"] = sq.RotaryPositions(config)
    empty = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    if case["kind"] == "rope":
        state["out"] = empty(case["rows"], case["heads"] * case["dim"])
        return state
    fmt = {"bf16": sq.KV_BF16, "int8": sq.KV_INT8, "e4m3": sq.KV_E4M3}[case["fmt"]]
    shape = sq.KvShape(kv_heads=case["kv_heads"], head_dim=case["dim"], page_rows=case["page"], format=fmt)
    state["cache"] = sq.kv_cache(shape, d["pages"], d["keys"], d["values"], d["key_scales"], d["value_scales"])
    state["batch"] = sq.kv_batch(d["starts"], d["lengths"], d["table"], d["rows"])
    if case["kind"] == "cache":
        state["k"], state["v"] = (empty(d["rows"], case["kv_heads"] * case["dim"]) for _ in range(2))
        state["q"] = empty(d["rows"], case["heads"] * case["dim"]) if case["rope"] else None
    else:
        attention = sq.AttentionShape(heads=case["heads"], kv=shape, window=case["window"], causal=1,
                                      scale=1 / math.sqrt(case["dim"]))
        state["plan"] = sq.attention_plan(attention, case["sequences"], d["rows"], max(r for r, _ in d["sizes"]))
        state["scratch"] = sq.AttentionScratch(state["plan"])
        state["out"] = empty(d["rows"], case["heads"] * case["dim"])
    return state


# ---------------------------------------------------------------- passes

def run(state):
    return run_own(state) if own else run_plain(state)


def run_own(state):
    sq, case, d = state["sq"], state["case"], state["d"]
    if case["kind"] == "rope":
        sq.rope_add(state["rope"], d["positions"], d["x"], state["out"], case["dim"])
        return state["out"]
    if case["kind"] == "attention":
        sq.attention_add(state["plan"], state["cache"], state["batch"], d["q"], state["out"], state["scratch"])
        return state["out"]
    if not case["read_only"]:
        q, kv = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
        x = d["qkv"]
        if case["rope"]:
            sq.kv_write(state["cache"], state["batch"], x[:, q:q + kv], x[:, q + kv:], rope=state["rope"],
                        queries=x[:, :q], rotated=state["q"])
        else:
            sq.kv_write(state["cache"], state["batch"], x[:, q:q + kv], x[:, q + kv:])
    sq.kv_read(state["cache"], state["batch"], state["k"], state["v"])
    return [state["k"], state["v"]] + ([state["q"]] if case["rope"] else [])


def rotate(x, positions, f, magnitude, layout):
    """x [rows, heads, dim] in fp32 with its first 2 len(f) dims rotated; angles in 64 bits."""
    angle = positions.double()[:, None] * f
    cos, sin = ((t(angle) * magnitude).float()[:, None] for t in (torch.cos, torch.sin))
    n = f.numel()
    out = x.clone()
    a, b = (x[..., :n], x[..., n:2 * n]) if layout == "half" else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    first, second = a * cos - b * sin, b * cos + a * sin
    if layout == "half":
        out[..., :n], out[..., n:2 * n] = first, second
    else:
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = first, second
    return out


def slots(d, case):
    """(page, row in it) of each of the batch's rows."""
    pages, rows = [], []
    for s, (n, keys) in enumerate(d["sizes"]):
        p = torch.arange(keys - n, keys, device="cuda")
        pages.append(d["table"][s, p // case["page"]].long())
        rows.append(p % case["page"])
    return torch.cat(pages), torch.cat(rows)


def run_plain(state):
    case, d = state["case"], state["d"]
    if case["kind"] == "rope":
        x = d["x"].float().reshape(case["rows"], case["heads"], case["dim"])
        y = rotate(x, d["positions"], state["frequencies"], state["magnitude"], case["layout"])
        return y.reshape(case["rows"], -1).to(torch.bfloat16)
    if case["kind"] == "attention":
        return attend_plain(case, d)
    rows, dim, kv = d["rows"], case["dim"], case["kv_heads"]
    page, slot = slots(d, case)
    rotated = []
    if not case["read_only"]:
        x = d["qkv"].float().reshape(rows, -1, dim)
        q, k, v = x.split([case["heads"], kv, kv], 1)
        if case["rope"]:
            positions = torch.cat([torch.arange(n - r, n, device="cuda") for r, n in d["sizes"]])
            turn = lambda t: rotate(t, positions, state["frequencies"], state["magnitude"], "half")  # noqa: E731
            rotated, k = [turn(q).reshape(rows, -1).to(torch.bfloat16)], turn(k)
        for name, t in (("key", k), ("value", v)):
            codes, scales = quantised(t, case["fmt"])
            d[name + "s"].view(torch.uint8 if case["fmt"] == "e4m3" else codes.dtype)[page, :, slot] = \
                codes.view(torch.uint8) if case["fmt"] == "e4m3" else codes
            if scales is not None:
                d[name + "_scales"][page, :, slot] = scales
    out = []
    for name in ("key", "value"):
        t = d[name + "s"]
        t = (t.view(torch.uint8)[page, :, slot].view(t.dtype) if case["fmt"] == "e4m3" else t[page, :, slot]).float()
        if case["fmt"] != "bf16":
            t = t * d[name + "_scales"][page, :, slot][..., None]
        out.append(t.reshape(rows, -1).to(torch.bfloat16))
    return out + rotated


def attend_plain(case, d):
    dim, kv, group = case["dim"], case["kv_heads"], case["heads"] // case["kv_heads"]
    out, at = [], 0
    for s, (n, keys) in enumerate(d["sizes"]):
        pages = d["table"][s, :-(-keys // case["page"])].long()

        def cached(name):
            t = d[name + "s"]
            t = t.view(torch.uint8)[pages].view(t.dtype) if case["fmt"] == "e4m3" else t[pages]
            t = t.float()
            if case["fmt"] != "bf16":
                t = t * d[name + "_scales"][pages][..., None]
            return t.transpose(0, 1).reshape(kv, -1, dim)[:, :keys]

        q = d["q"][at:at + n].float().reshape(n, kv, group, dim).permute(1, 2, 0, 3).reshape(kv, group * n, dim)
        scores = torch.bmm(q, cached("key").transpose(1, 2).contiguous()) * (1 / math.sqrt(dim))
        row, key = torch.arange(keys - n, keys, device="cuda")[:, None], torch.arange(keys, device="cuda")
        hidden = key > row
        if case["window"]:
            hidden = hidden | (key <= row - case["window"])
        scores = scores.reshape(kv, group, n, keys).masked_fill_(hidden, -math.inf)
        weights = torch.exp_(scores.sub_(scores.amax(-1, keepdim=True)))
        total = weights.sum(-1, keepdim=True)
        o = torch.bmm(weights.reshape(kv, group * n, keys), cached("value")).reshape(kv, group, n, dim) / total
        out.append(o.permute(2, 0, 1, 3).reshape(n, -1).to(torch.bfloat16))
        at += n
    return torch.cat(out)


# ---------------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    d = inputs(case, seed)
    if case["kind"] == "rope":
        return exact_rope(d["x"].reshape(case["rows"], -1, case["dim"]), d["positions"], case).flatten(1)
    if case["kind"] == "cache":
        return exact_cache(case, d)
    return exact_attention(case, d)


def exact_rope(x, positions, case):
    """Each pair as a complex number, turned by its angle."""
    f, magnitude = frequencies(case)
    d = case["rotary"]
    turn = torch.polar(torch.full((1, 1), magnitude, dtype=torch.float64, device="cuda"),
                       positions.double()[:, None] * f.cuda()[None])[:, None]
    x = x.double()
    head, tail = x[..., :d], x[..., d:]
    if case["layout"] == "half":
        z = turn * torch.complex(*head.chunk(2, -1))
        head = torch.cat([z.real, z.imag], -1)
    else:
        z = turn * torch.complex(head[..., 0::2].contiguous(), head[..., 1::2].contiguous())
        head = torch.view_as_real(z).flatten(-2)
    return torch.cat([head, tail], -1)


E4M3 = sorted({s * v for s in (-1.0, 1.0) for v in
               [m * 2.0 ** -9 for m in range(8)] +
               [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if not (e == 15 and m == 7)]})


def nearest(q, fmt):
    """The values of the 8-bit format nearest to q, ties to the even code."""
    if fmt == "int8":
        return torch.round(q)
    grid = torch.tensor(E4M3, dtype=torch.float64, device="cuda")
    above = torch.searchsorted(grid, q).clamp(1, grid.numel() - 1)
    lo, hi = grid[above - 1], grid[above]
    # 253 values, zero (code 0, even) at index 126: a code's last bit is that of its distance from there.
    even = torch.where((above - 1 - 126) % 2 == 0, lo, hi)
    return torch.where(q - lo < hi - q, lo, torch.where(q - lo > hi - q, hi, even))


def exact_cache(case, d):
    rows, dim, kv, heads = d["rows"], case["dim"], case["kv_heads"], case["heads"]
    if case["read_only"]:
        out = []
        for values, scales in (("keys", "key_scales"), ("values", "value_scales")):
            parts = []
            for s, (n, keys) in enumerate(d["sizes"]):
                for p in range((keys - n) // case["page"], -(-keys // case["page"])):
                    at = int(d["table"][s, p])
                    t = d[values][at].double()
                    if d[scales] is not None:
                        t = t * d[scales][at].double()[..., None]
                    lo, hi = max(0, keys - n - p * case["page"]), min(case["page"], keys - p * case["page"])
                    parts.append(t[:, lo:hi].transpose(0, 1))
            out.append(torch.cat(parts).flatten(1))
        return out
    x = d["qkv"].reshape(rows, heads + 2 * kv, dim)
    q, k, v = x[:, :heads], x[:, heads:heads + kv].double(), x[:, heads + kv:].double()
    extra = []
    if case["rope"]:
        positions = torch.cat([torch.arange(keys - n, keys, device="cuda") for n, keys in d["sizes"]])
        extra = [exact_rope(q, positions, rope_case(case)).flatten(1)]
        k = exact_rope(k, positions, rope_case(case))
    out = []
    for t in (k, v):
        if case["fmt"] != "bf16":
            top, largest = LARGEST[case["fmt"]], t.abs().amax(-1, keepdim=True)
            t = torch.where(largest > 0, nearest(t * top / largest, case["fmt"]) * (largest / top), 0.0)
        out.append(t.flatten(1))
    return out + extra


def exact_attention(case, d):
    dim, kv = case["dim"], case["kv_heads"]
    group, page = case["heads"] // kv, case["page"]
    out = torch.empty((d["rows"], case["heads"], dim), dtype=torch.float64, device="cuda")
    at = 0
    for s, (n, keys) in enumerate(d["sizes"]):
        position = torch.arange(keys, device="cuda")
        where, slot = d["table"][s].long()[position // page], position % page
        rows = torch.arange(keys - n, keys, device="cuda")
        allowed = position[None] <= rows[:, None]
        if case["window"]:
            allowed &= position[None] > rows[:, None] - case["window"]
        for h in range(kv):
            k, v = (t.view(torch.uint8)[where, h, slot].view(t.dtype).double() if case["fmt"] == "e4m3"
                    else t[where, h, slot].double() for t in (d["keys"], d["values"]))
            if case["fmt"] != "bf16":
                k = k * d["key_scales"][where, h, slot].double()[:, None]
                v = v * d["value_scales"][where, h, slot].double()[:, None]
            for g in range(group):
                head = h * group + g
                q = d["q"][at:at + n].reshape(n, -1, dim)[:, head].double()
                logits = (q @ k.T) / math.sqrt(dim)
                logits[~allowed] = -math.inf
                out[at:at + n, head] = torch.softmax(logits, -1) @ v
        at += n
    return out.flatten(1)
