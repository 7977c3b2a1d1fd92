"""The cache and attention operators at the ends of what a cache may be: 1024 heads, pages of 65536 positions and of thousands, a pool of a single
page, 128 query heads to a key / value head, thousands of sequences."""
import numpy as np
import pytest

import test_attn_decode as dec
import test_attn_prefill as pre
import test_kv_append as app
from attncase import BF16, F16, F32, Case

pytestmark = pytest.mark.gpu

CASES = [
    # type, t, n_q, n_kv, hd, page, lens, new, spare
    (F16, F32, 1024, 1024, 64, 16, (40, 3, 0, 17), (2, 2, 2, 2), 2),
    (BF16, BF16, 1024, 1024, 64, 16, (33,), (1,), 0),
    (F16, F16, 4, 1, 64, 65536, (66000, 90), (3, 3), 0),
    (BF16, F32, 2, 1, 128, 65536, (65536, 65537), (2, 2), 0),
    (F16, F32, 3, 1, 256, 4096, (5000, 4096, 4097), (1, 1, 1), 1),
    (F16, F32, 6, 2, 128, 1024, (1000,), (5,), 0),  # one page is the pool
    (BF16, BF16, 128, 1, 256, 32, (70, 1), (1, 1), 0),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_sizes(dev, i):
    ty, t, n_q, n_kv, hd, page, lens, new, spare = CASES[i]
    print(CASES[i], flush=True)
    c = Case(dev, 900 + i, ty, n_q, n_kv, hd, page, lens, new, spare=spare).fill_all().upload()
    print("decode", flush=True)
    dec.Call(c, t, new[0]).launch().check()
    print("prefill", flush=True)
    pre.Call(c, t).launch().check()
    pre.Call(c, t, window=100).launch().check()
    print("append", flush=True)
    app.check(c, t, 2, 64, app.run(c, t, 2, 64))


def test_sequences(dev):
    """5000 sequences, some of no rows and some of no part: a row's sequence is found in three steps of 64."""
    n = 5000
    lens = tuple(0 if i % 11 == 3 else 3 + i * 7 % 23 for i in range(n))
    new = tuple(i % 4 if lens[i] else i % 3 for i in range(n))
    c = Case(dev, 920, F16, 2, 1, 64, 16, lens, new, room=9).fill_all().upload()
    print("prefill", flush=True)
    pre.Call(c, F16).launch().check()
    print("append", flush=True)
    app.check(c, F32, 1, 64, app.run(c, F32, 1, 64))
    print("decode", flush=True)
    c = Case(dev, 921, F16, 2, 1, 64, 16, lens, (2,) * n).fill_all().upload()
    dec.Call(c, F32, 2).launch().check()
