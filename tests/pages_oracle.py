"""A pool of cache pages on the host (numpy): its books and bytes, and what each call makes of them, one request after the
other."""
from __future__ import annotations

import numpy as np

import splash_q4 as sq
from cache4_oracle import scale_bytes

HOLE = 0xFFFFFFFF
FORMATS = {"bf16": sq.KV_BF16, "int8": sq.KV_INT8, "e4m3": sq.KV_E4M3, "e2m1": sq.KV_E2M1}


def torch():
    import torch as t
    return t


def row_bytes(fmt, dim):
    """Bytes of a head row's values and scale."""
    return {"bf16": (2 * dim, 0), "int8": (dim, 4), "e4m3": (dim, 4), "e2m1": (dim // 2, scale_bytes(dim))}[fmt]


class Pool:
    """Books and bytes: pools[i] is [pages, kv_heads, page_rows, bytes] of keys, values, key scales, value scales."""

    def __init__(self, rng, pages, sequences, pages_per_sequence, kv_heads=2, dim=64, page=16, fmt="int8"):
        self.shape = sq.KvShape(kv_heads, dim, page, FORMATS[fmt])
        self.pages, self.page, self.fmt = pages, page, fmt
        self.references = np.zeros(pages, np.uint32)
        self.table = np.full((sequences, pages_per_sequence), HOLE, np.uint32)
        self.lengths = np.zeros(sequences, np.uint32)
        self.report = np.zeros(4, np.uint32)
        value, scale = row_bytes(fmt, dim)
        self.pools = [rng.integers(0, 256, (pages, kv_heads, page, n), dtype=np.uint8)
                      for n in (value, value, scale, scale)]

    # ---- what the calls do

    def free(self):
        return list(np.flatnonzero(self.references == 0))

    def copy_rows(self, source, target, rows):
        for p in self.pools:
            p[target][:, :rows] = p[source][:, :rows]

    def release(self, rows, keeps):
        self.report[:2] = sum(int(r >= len(self.lengths)) for r in rows), 0
        for r, keep in zip(rows, keeps):
            if r >= len(self.lengths):
                continue
            self.lengths[r] = min(self.lengths[r], keep)
            for e in range(-(-int(keep) // self.page), self.table.shape[1]):
                page = self.table[r, e]
                if page < self.pages and self.references[page]:
                    self.references[page] -= 1
                self.table[r, e] = HOLE

    def take(self, rows, parents, more):
        """A grow (parents None) or a fork (more None)."""
        fork, seen, free, wanted, lost, copied = more is None, set(), self.free(), 0, 0, 0
        copies, drops, gains = [], [], []
        for i, r in enumerate(rows):
            parent = int(parents[i]) if fork else int(r)
            ok = r < len(self.lengths) and parent < len(self.lengths) and r not in seen and not (fork and r in parents)
            seen.add(r)
            new = []
            if ok:
                keys = min(int(self.lengths[parent]), self.table.shape[1] * self.page)
                grown = keys if fork else keys + int(more[i])
                ok = grown <= self.table.shape[1] * self.page
            if ok:
                full, part = divmod(keys, self.page)
                last = self.table[parent, full] if part else HOLE
                copy = last < self.pages and (fork or (grown > keys and self.references[last] > 1))
                entries = [full] if copy else []
                if not fork:
                    entries += range(full + (part > 0), -(-grown // self.page))
                wanted += len(entries)
                ok = not entries or wanted <= len(free)
            if not ok:
                lost += 1
                continue
            new = free[wanted - len(entries):wanted]
            if fork:
                for e in range(self.table.shape[1]):
                    page = self.table[parent, e] if e < full else HOLE
                    if page < self.pages:
                        gains.append(page)
                    self.table[r, e] = page if page < self.pages else HOLE
            for e, page in zip(entries, new):
                self.table[r, e] = page
                gains.append(page)
            if copy:
                copied += 1
                copies.append((int(last), int(new[0]), part))
                if not fork:
                    drops.append(last)
            self.lengths[r] = grown
        for page in gains:
            self.references[page] += 1
        for page in drops:
            self.references[page] -= 1
        for c in copies:
            self.copy_rows(*c)
        self.report[:2] = lost, copied

    def fork(self, parents, children):
        self.take(children, parents, None)

    def grow(self, rows, more):
        self.take(rows, None, more)

    def compact(self):
        used, free = np.flatnonzero(self.references), np.flatnonzero(self.references == 0)
        live = len(used)
        to = free[free < live]
        source = used[::-1][:len(to)]
        place = {}
        for a, b in zip(source, to):
            self.copy_rows(a, b, self.page)
            self.references[b], self.references[a] = self.references[a], 0
            place[a] = b
        for index, page in np.ndenumerate(self.table):
            self.table[index] = place.get(page, page)
        self.report[:3] = 0, len(to), live

    def check_books(self):
        named = self.table[self.table < self.pages]
        assert np.array_equal(np.bincount(named, minlength=self.pages), self.references)


class DevicePool:
    """The same on the device, and the library's calls on it; guards of a word lie on both sides of every view."""

    def __init__(self, pool: Pool):
        t = torch()
        self.host = pool
        self.guarded = []

        def put(array):
            flat = np.ascontiguousarray(array).view(np.uint8).reshape(-1)
            whole = t.full((64 + flat.size + 64,), 0xA5, dtype=t.uint8, device="cuda")
            whole[64:64 + flat.size] = t.from_numpy(flat.copy()).cuda()
            self.guarded.append(whole)
            return whole[64:64 + flat.size]

        self.pools = [put(p) if p.size else None for p in pool.pools]
        words = lambda a: put(a).view(t.int32)  # noqa: E731
        self.references, self.lengths, self.report = words(pool.references), words(pool.lengths), words(pool.report)
        self.table = words(pool.table).view(*pool.table.shape)
        self.cache = sq.kv_cache(pool.shape, pool.pages, *(p if p is None or i < 2 or pool.fmt == "e2m1" else p.view(t.float32)
                                                           for i, p in enumerate(self.pools)))
        self.struct = sq.kv_pool(self.cache, self.references, self.table, self.lengths, self.report)
        self.scratch = sq.KvPoolScratch(self.struct)
        self.scratch.workspace.fill_(0xFF)

    def words(self, values):
        return torch().from_numpy(np.asarray(values, np.uint32).view(np.int32)).cuda()

    def release(self, rows, keeps):
        sq.kv_release(self.struct, self.words(rows), self.words(keeps))

    def grow(self, rows, more):
        sq.kv_grow(self.struct, self.words(rows), self.words(more), self.scratch)

    def fork(self, parents, children):
        sq.kv_fork(self.struct, self.words(parents), self.words(children), self.scratch)

    def compact(self):
        sq.kv_compact(self.struct, self.scratch)

    def state(self):
        torch().cuda.synchronize()
        get = lambda x: x.cpu().numpy().view(np.uint32)  # noqa: E731
        return {"references": get(self.references), "table": get(self.table), "lengths": get(self.lengths),
                "report": get(self.report)}

    def check(self, what=""):
        got = self.state()
        for name, x in got.items():
            want = getattr(self.host, name)
            assert np.array_equal(x, want), f"{what}: {name} at {np.argwhere(x != want)[:5].tolist()}"
        for got_p, want_p in zip(self.pools, self.host.pools):
            if got_p is not None:
                same = got_p.cpu().numpy().reshape(want_p.shape) == want_p
                assert same.all(), f"{what}: bytes at {np.argwhere(~same)[0].tolist()}"
        self.check_guards()

    def check_guards(self):
        for whole in self.guarded:
            assert (whole[:64] == 0xA5).all() and (whole[-64:] == 0xA5).all()
