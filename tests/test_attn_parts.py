"""The f32 accuracy of f32 queries: every 16-bit part of the queries and of the weights reaches the products (f16 caches: two parts each, bf16
three), in every kernel that takes f32 queries. The inputs are such that a lost part shows as an error far over the bound, which the CPU
tests show by losing one.

Queries: value pairs (2 i, 2 i + 1) of a query are c + a 2^-b and c, a in 0 .. 3, and the keys that count are 1, -1 in one pair and 0
elsewhere: their products, a 2^-b, are exact, and what the part that holds a 2^-b loses is all of it. With scale 2^b their scores are a.
Weights: a row sees two positions that count, values 1 and -1, whose scores, exact, are under 1/2 apart: y = (u - w) / (u + w), so that an
error of a weight is one of y at half its size. All other positions have scores so low that their weights are 0."""
import numpy as np
import pytest

import test_attn_decode as dec
import test_attn_prefill as pre
from attncase import BF16, F16, F32, Case, attn64, from16, to16

# Queries: scores of at most 3, 4.4 in base 2. The scale times log2(e), a product of it and the sum with the reference (8 at most more, a
# result of 16 at most) are rounded once each: 4.4 x 2 2^-24 + 2 2^-21 (half a step of results under 16) and as much for the reference, with
# the exponential's 2^-23 a factor of 1 + 2^-18.9 at most of a weight; the joins' exponentials of differences under 4.4 twice 2^-22. In the
# weighted and the plain sum: 2^-17 of sum w |v| / sum w; |v| is under 8.
QUERIES = 2.0 ** -14
# Weights: arguments of the exponential between -0.8 and 0 (f16: 7.2 and 8) are off by 1.75 2^-24 (2^-22 + 1.5 2^-24), a weight so by a factor of
# 1.2 2^-24 (2^-22), by the exponential's 2^-23 and by its parts' 2^-27 (2^-24); y by half the two weights' sum, and by six roundings of the sums
# and the division, of values half as large: under 7 2^-24 (under 2.5 2^-22).
WEIGHTS = {BF16: 2.0 ** -21, F16: 2.0 ** -20}
FULL = {F16: 2, BF16: 3}
# c and b: which part of the queries holds a 2^-b (bf16 parts: 8 bits each; f16: 11)
LEVELS = {F16: [(1.0, 21)], BF16: [(1.0, 12), (1.0 + 2.0 ** -9, 23)]}


def split(x, ty, n):
    """x as the sum of its first n parts."""
    x = np.asarray(x, np.float64)
    got = np.zeros_like(x)
    for _ in range(n):
        got += from16(to16((x - got).astype(np.float32), ty), ty).reshape(x.shape)
    return got


def of_queries(dev, seed, ty, n_q, n_kv, hd, lens, new, level, page=16):
    """A case and its queries."""
    c0, b = LEVELS[ty][level]
    c = Case(dev, seed, ty, n_q, n_kv, hd, page, lens, new)
    rows = sum(new)
    q = np.full((rows, n_q, hd), c0)
    q[:, :, 0::2] += c.g.integers(0, 4, (rows, n_q, hd // 2)) * 2.0 ** -b
    for s, (L, m) in enumerate(zip(lens, new)):
        c.k[s][:] = 0
        c.k[s][:, :, 0] = -1  # a score of -2^b
        at = np.unique(np.linspace(0, L - m, hd // 2).astype(int))
        for i, p in enumerate(at):
            c.k[s][p] = 0
            c.k[s][p, :, 2 * i], c.k[s][p, :, 2 * i + 1] = 1, -1
    return c.fill_all(), q, 2.0 ** b


def of_weights(dev, seed, ty, n_q, n_kv, hd, lens, new, page=16):
    """A case, its queries, and for each sequence its first position that counts (the second is the next)."""
    c = Case(dev, seed, ty, n_q, n_kv, hd, page, lens, new)
    G, rows = n_q // n_kv, sum(new)
    q = np.zeros((rows, n_q, hd))
    r, h = np.meshgrid(np.arange(rows), np.arange(n_q), indexing="ij")
    q[r, h, (7 * (h % G) + 13 * r + 5 * (h // G)) % hd] = 1
    first = []
    for s, (L, m) in enumerate(zip(lens, new)):
        p = (L - m) * (s + 1) // (len(lens) + 1) & ~1  # in the middle, or near an end
        first.append(p)
        c.k[s][:] = -200
        c.k[s][p:p + 2] = -0.5 * c.g.random((2, n_kv, hd))
        c.v[s][p], c.v[s][p + 1] = 1, -1
    return c.fill_all(), q, first


def two(q, k, first, ty, nq, nw):
    """y of a row of one head over the two positions, in 64 bits, the query in nq and the weights in nw parts."""
    s = k[first:first + 2] @ split(q, ty, nq)
    w = split(np.exp(s - s.max()).astype(np.float32), ty, nw)
    return (w[0] - w[1]) / w.sum()


@pytest.mark.parametrize("ty,level", [(F16, 0), (BF16, 0), (BF16, 1)])
def test_a_lost_part_of_queries_shows(ty, level):
    c, q, scale = of_queries(None, 3, ty, 4, 2, 64, (300,), (2,), level)
    k, v = c.stored(0)
    want = attn64(q, k, v, scale, np.array([298, 299]), 0)[0]
    for n in range(1, FULL[ty] + 1):
        off = np.abs(attn64(split(q, ty, n), k, v, scale, np.array([298, 299]), 0)[0] - want).max()
        # the part that holds a 2^-b is the last one that counts: with it the queries are whole
        assert off == 0 if n >= (level + 2) else off > 1000 * QUERIES


@pytest.mark.parametrize("ty", (F16, BF16))
def test_a_lost_part_of_weights_shows(ty):
    c, q, first = of_weights(None, 5, ty, 24, 2, 64, (70, 400), (2, 2))
    for n in range(1, FULL[ty] + 1):
        off = 0.0
        for s in range(2):
            k, _ = c.stored(s)
            for r in range(2 * s, 2 * s + 2):
                for h in range(24):
                    args = q[r, h], k[:, h // 12], first[s], ty
                    off = max(off, abs(two(*args, 1, n) - two(*args, 1, 9)))
        assert off < WEIGHTS[ty] / 4 if n == FULL[ty] else off > 4 * WEIGHTS[ty], (n, off)


# n_q, n_kv, T: up to 16 columns, and blocks of 32 (heads of up to 128)
DECODE = [(hd, n_q, n_kv, T) for hd in (64, 128, 256) for n_q, n_kv, T in ((12, 2, 2), (28, 4, 5))]


def name(hd, ty, tail=""):
    return f"h{hd}_{'f16' if ty == F16 else 'bf16'}_f32{tail}"


def check(y, want, av, tol):
    off = np.abs(y - want) / tol
    assert off.max() <= 1, f"{off.max():.2f} of the bound, {int((~(off <= 1)).sum())} values"


def queries(dev, op, c, q, scale, window=0):
    a = dec.Call(c, F32, c.new[0], q=q, scale=scale, window=window) if op == "decode" else pre.Call(c, F32, q=q, scale=scale, window=window)
    y, r0 = a.launch().got(), 0
    kernel = dev.last_kernel()
    for s, (L, m) in enumerate(zip(c.lens, c.new)):
        k, v = c.stored(s)
        assert np.abs(v).max() < 8
        want, av, _ = attn64(q[r0:r0 + m], k, v, scale, np.arange(L - m, L), window)
        check(y[r0:r0 + m], want, av, QUERIES)
        r0 += m
    return kernel


def weights(dev, op, c, q, first, tol):
    a = dec.Call(c, F32, c.new[0], q=q, scale=1.0) if op == "decode" else pre.Call(c, F32, q=q, scale=1.0)
    y, r0 = a.launch().got(), 0
    for s, (L, m) in enumerate(zip(c.lens, c.new)):
        k, v = c.stored(s)
        want, av, _ = attn64(q[r0:r0 + m], k, v, 1.0, np.arange(L - m, L), 0)
        check(y[r0:r0 + m], want, av, tol)
        r0 += m
    return dev.last_kernel()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", (F16, BF16))
@pytest.mark.parametrize("hd,n_q,n_kv,T", DECODE)
def test_decode(dev, ty, hd, n_q, n_kv, T):
    """Sequences within a step, of one chunk and of several."""
    kernel = "amdc_attn_dec_" + name(hd, ty, "_n2" if T * n_q // n_kv > 16 and hd <= 128 else "")
    for level in range(len(LEVELS[ty])):
        c, q, scale = of_queries(dev, 800 + hd, ty, n_q, n_kv, hd, (25, 333, 6000), (T, T, T), level)
        assert queries(dev, "decode", c.upload(), q, scale) == kernel
    c, q, first = of_weights(dev, 810 + hd, ty, n_q, n_kv, hd, (25, 333, 6000, 6100), (T, T, T, T))
    assert weights(dev, "decode", c.upload(), q, first, WEIGHTS[ty]) == kernel


@pytest.mark.gpu
@pytest.mark.parametrize("ty", (F16, BF16))
@pytest.mark.parametrize("hd", (64, 128, 256))
def test_prompts(dev, ty, hd):
    """Tiles that all rows see and ones at the edge, split over the positions or not."""
    for lens, new in (((239, 90, 60), (40, 20, 2)), ((4000, 239, 1500), (30, 40, 5))):
        split_up = lens[0] > 1000
        kernel = "amdc_attn_join_f32" if split_up else "amdc_attn_pre_" + name(hd, ty)
        for level in range(len(LEVELS[ty])):
            c, q, scale = of_queries(dev, 820 + hd, ty, 6, 2, hd, lens, new, level)
            assert queries(dev, "prefill", c.upload(), q, scale) == kernel
        c, q, first = of_weights(dev, 830 + hd, ty, 6, 2, hd, lens, new)
        assert weights(dev, "prefill", c.upload(), q, first, WEIGHTS[ty]) == kernel
