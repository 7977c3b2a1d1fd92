"""Rows that are NaN: a page that cannot be followed, a key that is NaN, a scale that is NaN, in both attention operators, as y and as the
Q8 copy, which is amdc_quant_q8's of the f32 result there too (a block that is all NaN has d = NaN, so that the matrix product that reads it
is NaN as well)."""
import numpy as np
import pytest

import test_attn_decode as dec
import test_attn_prefill as pre
from attncase import BF16, F16, F32, Case

pytestmark = pytest.mark.gpu
NAN = {F16: 0x7E01, BF16: 0x7FC1}


def quantized(dev, y):
    """amdc_quant_q8's bytes of rows y (f32)."""
    rows, w = y.shape
    xs = w // 32 * 40
    X, Q = dev.DevBuf.of(y), dev.DevBuf(rows * xs)
    dev.quant_q8(X, Q, w // 32, rows, 4 * w, xs)
    dev.sync()
    return Q.download(np.uint8).reshape(rows, xs)


def parts(q, w):
    """The q, d and sums of Q8 rows."""
    nb = w // 32
    q = np.ascontiguousarray(q)
    return q[:, :w], q[:, w:w + 4 * nb].copy().view(np.float32), q[:, w + 4 * nb:w + 8 * nb].copy().view(np.uint32)


def run(dev, op, c, t, T):
    """(y, its Q8 copy, the copy without y) of the call's rows."""
    a = dec.Call(c, t, T, q8=True) if op == "decode" else pre.Call(c, t, q8=True)
    a.launch()
    y = a.got().reshape(a.rows, a.w)
    q = a.Q8.download(np.uint8).reshape(a.rows, a.q8s)
    a.Q8.fill(0xA5)
    if op == "decode":
        a.Y = None
        a.launch()
    else:
        a.launch(y=False)
    dev.sync()
    return y.astype(np.float32), q, a.Q8.download(np.uint8).reshape(a.rows, a.q8s)


def check(dev, y, q, again, bad):
    w = y.shape[1]
    assert np.isnan(y[bad]).all() and np.isfinite(y[~bad]).all()
    want = parts(quantized(dev, y), w)
    for got in (parts(q, w), parts(again, w)):
        assert np.isnan(got[1][bad]).all(), "a row that is NaN reads as a number in its Q8 copy"
        for g, x in zip(got, want):
            assert np.array_equal(g, x, equal_nan=g.dtype == np.float32)


# type, n_q, n_kv, hd, lens, new: prompts that are not split over their positions, and ones that are
PROMPTS = [(F16, 4, 2, 64, (90, 50), (20, 9)), (BF16, 4, 2, 128, (90, 50), (90, 9)), (F16, 4, 2, 256, (90, 50), (20, 9)),
           (F16, 4, 2, 64, (2000, 50), (20, 9)), (BF16, 4, 2, 128, (2000, 50), (20, 9)), (F16, 4, 2, 256, (2000, 50), (20, 9))]


@pytest.mark.parametrize("i", range(len(PROMPTS)))
@pytest.mark.parametrize("what", ("page", "key"))
def test_prompts(dev, i, what):
    ty, n_q, n_kv, hd, lens, new = PROMPTS[i]
    c = Case(dev, 700 + i, ty, n_q, n_kv, hd, 16, lens, new).fill_all()
    if what == "page":
        c.table[0, 2] = 999
    else:
        c.K[c.table[0, 2], :, 0, 0, 1, 3] = NAN[ty]  # position 33
    c.upload()
    y, q, again = run(dev, "prefill", c, F32, None)
    assert ("join" in dev.last_kernel()) == (lens[0] > 1000), "split or not, as the case is meant to be"
    bad = np.zeros(sum(new), bool)
    bad[:new[0]] = lens[0] - new[0] + np.arange(new[0]) >= 33
    if what == "page":
        with pytest.raises(dev.AmdcError, match="page outside"):
            dev.kv_check()
        # which rows before the page's positions are NaN as well is open: those of the tile; here only the others are compared
        bad[:new[0]] |= np.isnan(y[:new[0]]).all(1)
    check(dev, y, q, again, bad)


@pytest.mark.parametrize("ty,n_q,hd,T", [(F16, 4, 64, 2), (BF16, 4, 128, 2), (F16, 4, 256, 2), (F16, 24, 128, 3)])
@pytest.mark.parametrize("n", (90, 4000))
@pytest.mark.parametrize("what", ("page", "key", "length"))
def test_decode(dev, ty, n_q, hd, T, n, what):
    c = Case(dev, 720 + hd + T, ty, n_q, 2, hd, 16, (n, 50), (T, T)).fill_all()
    if what == "page":
        c.table[0, 2] = 999
    elif what == "key":
        c.K[c.table[0, 2], :, 0, 0, 1, 3] = NAN[ty]
    c.upload()
    if what == "length":
        c.dlen.upload(np.array([5 * n, 50], np.int32))
    y, q, again = run(dev, "decode", c, F32, T)
    if what != "key":
        with pytest.raises(dev.AmdcError, match="page outside" if what == "page" else "length"):
            dev.kv_check()
    check(dev, y, q, again, np.repeat([True, False], T))
