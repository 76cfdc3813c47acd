"""The weights of the attention's tiles of 16 and 32 rows enter the second product as two bf16 each: outputs are held to a
bound that one bf16 a weight does not keep, which the first tests here show by arithmetic alone."""
import math

import numpy as np
import pytest

import splash_q4 as sq
from attention_oracle import FORMATS, HALF_STEP, Cache, bf16, run_attention

# A weight in [2^e, 2^(e+1)) rounded down leaves less than 2^(e-7), whose rounding to bf16 is off by half of 2^(e-15) at most:
# 2^-16 of the weight. All weights grow by 2^-18 on their way in.
TWO = 2.0 ** -16 + 2.0 ** -18


def attend(x, k, v, scale, enter=lambda p: p):
    """(outputs, their bounds) of query rows x [n, dim] that see all keys k, v [keys, dim]. enter: what becomes of a weight
    in the second product.

    The bound: an output's own rounding, the weights' (TWO of sum p |v|), and fp32 sums: a score is off by (dim + 4) 2^-24
    sum |q k| scale and its exponential by 2^-22 of the score, in both directions within the sums; weights, products (two
    a weight) and the quotient by 2^-24 each in chains of keys / 16 + 64 at most."""
    dim, keys = x.shape[1], len(k)
    t = (x @ k.T) * scale
    p = np.exp(t - t.max(-1, keepdims=True))
    total = p.sum(-1, keepdims=True)
    o, size = enter(p) @ v / total, p @ np.abs(v) / total
    products = (np.abs(x) @ np.abs(k).T * abs(scale)).max(-1, keepdims=True)
    score = (dim + 4) * 2 ** -24 * products + 2 ** -22 * np.abs(t).max(-1, keepdims=True)
    slack = 2 * np.expm1(score) + (keys / 16 + 64) * 2 ** -24
    return o, HALF_STEP * np.abs(o) + size * (TWO + slack) * (1 + HALF_STEP)


def down(p):
    """Positive fp32 values rounded down to bf16."""
    return (np.asarray(p, np.float32).view(np.uint32) & 0xFFFF0000).view(np.float32).astype(np.float64)


def one(p):
    return bf16(p)


def two(p):
    return down(p) + bf16(p * (1 + 2.0 ** -18) - down(p))


@pytest.mark.parametrize("dim,keys", [(64, 2), (128, 5), (256, 9), (64, 33), (128, 70)])
def test_the_bound_tells_one_rounding_from_two(dim, keys):
    rng = np.random.default_rng(dim + keys)
    x, k, v = (bf16(rng.standard_normal((n, dim)) * s) for n, s in ((4, 0.5), (keys, 0.3), (keys, 1.0)))
    want, bound = attend(x, k, v, 1 / math.sqrt(dim))
    for enter, holds in ((two, True), (one, False), (down, False)):
        got, _ = attend(x, k, v, 1 / math.sqrt(dim), enter)
        assert np.all(np.abs(bf16(got) - want) <= bound) == holds, enter.__name__


# One new row a sequence, of few keys whose weights are alike, so that no output is far above what a weight is off by.
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv_heads,dim,sizes,tile", [
    (4, 2, 64, [2, 3, 5, 9, 17, 33, 70], 16), (8, 1, 128, [2, 3, 7, 40, 130], 16), (8, 2, 256, [2, 5, 33, 90], 16),
    (2, 1, 80, [3, 64], 16), (20, 1, 64, [2, 3, 5, 33], 32), (32, 1, 128, [2, 5, 17, 70], 32), (8, 1, 128, [20001], 16),
])
def test_weights_of_few_rows(fmt, heads, kv_heads, dim, sizes, tile):
    rng = np.random.default_rng(heads + dim)
    c = Cache(rng, [(1, n) for n in sizes], kv_heads, dim, 16, fmt, key_scale=0.3).fill()
    plan = sq.attention_plan(sq.AttentionShape(heads, c.shape, 1, 0, 1 / math.sqrt(dim)), len(sizes), c.rows, 1)
    assert plan.tile_rows == tile
    q = bf16(rng.standard_normal((c.rows, heads, dim)) * 0.5)
    got = run_attention(c, q, 1 / math.sqrt(dim), plan=plan)
    group, missed = heads // kv_heads, 0
    for s in range(len(sizes)):
        k, v = c.stored(s)
        for h in range(kv_heads):
            x = q[s, h * group:(h + 1) * group]
            want, bound = attend(x, k[h], v[h], 1 / math.sqrt(dim))
            err = np.abs(got[s, h * group:(h + 1) * group] - want)
            assert np.all(err <= bound), (sizes[s], h, np.max(err / bound))
            missed += np.sum(np.abs(bf16(attend(x, k[h], v[h], 1 / math.sqrt(dim), one)[0]) - want) > bound)
    assert missed or sizes == [20001], "one rounding a weight would have kept the bound here"


@pytest.mark.parametrize("scale,fits", [(2.3e38, True), (-2.3e38, True), (2.4e38, False), (-3.4e38, False), (1e-45, True)])
def test_scales_whose_product_overflows(scale, fits):
    """The exponentials are of two, their arguments scale log2 e times the products: past fp32's range that is infinite, and
    a key that is not seen, or a product of zero, would come out as NaN."""
    shape = sq.AttentionShape(8, sq.KvShape(2, 64, 16, sq.KV_BF16), 1, 0, scale)
    if fits:
        sq.attention_plan(shape, 1, 1, 1)
    else:
        with pytest.raises(sq.InvalidArgument, match="scale"):
            sq.attention_plan(shape, 1, 1, 1)
