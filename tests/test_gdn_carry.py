"""amdc_gdn_prefill over more chunks than a pair of launches takes: a single sequence (with cu, from its first row or a later one, and
without), sequences of one length without cu, and packed ones, whose chunks go on from one pair of launches to the next; in place, from zeros,
into no slot. A state lost between two launches would be off by over 200 times the bound in the next one's first rows (the same sequences in 64 bits)."""
import numpy as np
import pytest

from attncase import BF16, F32, TINY, ULP, as_float
from lincase import near, state_of
from test_gdn_decode import Call
from test_gdn_prefill import some_heads

pytestmark = pytest.mark.gpu
N_K, N_V, DK, DV = 32, 128, 128, 16  # 6.4 MB a chunk
HEADS = [3, 100]


@pytest.fixture(scope="module")
def most(dev):
    """The chunks of a pair of launches: where the workspace stops growing with the rows."""
    g = dev.Gdn(N_K, N_V, DK, DV, 1, 0.1, 1e-6, dev.DevBuf(4), dev.DevBuf(4))
    size = lambda chunks: dev.gdn_prefill_ws(g, 1, 64 * (chunks - 1) + 1)
    lo, hi = 1, 1 << 14
    assert size(lo) < size(hi) == size(4 * hi)
    while hi - lo > 1:
        mid = (lo + hi) // 2
        lo, hi = (lo, mid) if size(mid) == size(4 << 14) else (mid, hi)
    assert 16 < hi < 200  # sequences below: of several launches, and small enough for the host
    return hi


def check(dev, new, t=BF16, skip=0, **kw):
    """skip: rows before the first sequence's."""
    c = Call(dev, 1600 + len(new), new, N_K, N_V, DK, DV, tiled=True, t=t, prefill=True, room=skip, **kw)
    s = c.s
    s.cu += np.int32(skip)
    if skip:  # the room is ahead of the sequences
        for a in (c.L.raw, c.L.x, c.L.ab):
            a[:] = np.roll(a, skip, 0)
    c.upload().launch()
    dev.kv_check()
    raw, pool = c.results()
    pool = state_of(pool.reshape(s.n_slots, N_V, DV // 16, DK, 16))
    y, L = as_float(raw, t).reshape(-1, N_V, DV)[:, HEADS], some_heads(c.L, HEADS)
    assert (raw[:skip] == 7).all()
    for b in range(s.n):
        old = c.S[s.start[b]][HEADS] if s.start[b] >= 0 else np.zeros((len(HEADS), DK, DV))
        want, err, st, es = L.run64(s.at(b), old, chunk=64)
        near(y[s.at(b)], want, err * (1 + ULP[t]) + ULP[t] * np.abs(want) + TINY[t], f"sequence {b}")
        if s.to[b] >= 0:
            near(pool[s.to[b]][HEADS].astype(np.float64), st[-1], es[-1], f"state {b}")
    others = [i for i in range(s.n_slots) if i not in s.to]
    assert np.array_equal(pool[others], c.S[others])


@pytest.mark.parametrize("how", ("cu", "cu from a later row", "no cu"))
@pytest.mark.parametrize("start,to", [((0,), (0,)), ((-1,), (1,)), ((1,), (-1,))])
def test_single(dev, most, how, start, to):
    """Over three pairs of launches, the last chunk not whole."""
    m = 64 * (2 * most + 1) + 37
    check(dev, (m,), ragged=how != "no cu", skip=64 * 3 + 5 if "later" in how else 0, start=start, to=to)


@pytest.mark.parametrize("t", (F32, BF16))
def test_one_length(dev, most, t):
    """Without cu, sequences that straddle the launches' ends: one and a bit to a launch, and many."""
    check(dev, (64 * (most - 9) + 5,) * 3, t, ragged=False, start=(2, -1, 0), to=(2, 1, -1))
    n = 2 * most // 3 + 5  # of 3 chunks: two pairs of launches
    check(dev, (150,) * n, t, ragged=False, start=[-1 if b % 3 == 0 else b for b in range(n)], to=[-1 if b % 5 == 1 else b for b in range(n)])


def test_ends(dev, most):
    """Packed: a sequence that ends with a launch, one that begins with the next, and ones that fill launches exactly."""
    check(dev, (64 * most, 64 * most, 64 * (most - 2), 64 * 2, 20), ragged=True, start=(0, -1, 2, 3, -1), to=(0, 1, 2, 3, 4))
