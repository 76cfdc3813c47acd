"""The cache's writes and reads of many rows, which take a wave a row where fewer have a workgroup: the bits of the same rows
in smaller calls, and of the definition."""
import numpy as np
import pytest

import splash_q4 as sq
from attention_oracle import FORMATS, Cache, bf16, from_bf16, quantised, to_bf16, torch

pytestmark = pytest.mark.gpu

FEW = 2048     # rows that have a workgroup each


def same(a, b):
    return torch().equal(a.view(torch().uint8), b.view(torch().uint8))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,interleaved", [
    (6, 2, 64, 64, False), (3, 3, 128, 100, True), (8, 1, 80, 20, False), (4, 2, 256, 256, False), (5, 5, 16, 6, False),
])
def test_many_rows_are_the_rows_of_smaller_calls(fmt, heads, kv_heads, dim, rotary, interleaved):
    """One call of 3400 rows (with a rope, queries beside the keys, rows of no sequence, rows before position 0 and pages that
    are holes) and the same sequences in calls of their own, under and at the border."""
    t = torch()
    sizes = [(FEW, 2500), (0, 40), (700, 650), (1, 77), (640, 640)]
    rope = sq.RotaryPositions(sq.RopeConfig(rotary_dim=rotary, layout=int(interleaved), base=1e4))
    one, many = (Cache(np.random.default_rng(1), sizes, kv_heads, dim, 32, fmt, extra_rows=11) for _ in range(2))
    for c in (one, many):
        c.table[0, 3], c.table[2, 0] = 0xFFFFFFFF, c.pages
        c.table_d.copy_(t.from_numpy(c.table.view(np.int32)))
    rng = np.random.default_rng(2)
    fused = to_bf16(bf16(rng.standard_normal((one.rows, (heads + 2 * kv_heads) * dim))))
    q, k, v = fused.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
    made = lambda width: t.full((one.rows, width * dim), 7.0, dtype=t.bfloat16, device="cuda")  # noqa: E731
    a, b = ([made(heads), made(kv_heads), made(kv_heads)] for _ in range(2))
    sq.kv_write(one.struct(), one.batch(), k, v, rope=rope, queries=q, rotated=a[0])
    sq.kv_read(one.struct(), one.batch(), a[1], a[2])
    for s, (n, _) in enumerate(sizes):
        if not n:
            continue
        at = slice(int(many.starts[s]), int(many.starts[s + 1]))
        starts = t.tensor([0, n], dtype=t.int32, device="cuda")
        batch = sq.kv_batch(starts, many.lengths_d[s:s + 1], many.table_d[s:s + 1], n)
        sq.kv_write(many.struct(), batch, k[at], v[at], rope=rope, queries=q[at], rotated=b[0][at])
        sq.kv_read(many.struct(), batch, b[1][at], b[2][at])
    t.cuda.synchronize()
    assert all(same(x, y) for x, y in zip(a, b))
    for name in ("keys", "values", "key_scales", "value_scales"):
        assert same(getattr(one, name), getattr(many, name)), name
    assert all((x[one.live_rows:] == 7).all() for x in a)
    # Values have no rope: theirs are the definition's.
    codes, scales = quantised(from_bf16(v.contiguous()).reshape(one.rows, kv_heads, dim), fmt)
    want = bf16(codes.astype(np.float32) * scales[..., None])
    first, got = int(one.starts[4]), from_bf16(a[2]).reshape(one.rows, kv_heads, dim)
    assert np.array_equal(got[first:one.live_rows], want[first:one.live_rows])
