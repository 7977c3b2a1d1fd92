"""amdc_gdn_prefill against the recurrence in 64 bits: lengths around the chunks of 64, ragged packing, all head sizes, types and
orders; states in place, shared, from zeros; sequences that go on from one pair of launches to the next; and that it agrees with
amdc_gdn_decode."""
import copy

import numpy as np
import pytest

from attncase import BF16, F16, F32, TINY, ULP, from16
from lincase import U, near, pool_of, state_of
from test_gdn_decode import HEADS, Call as Both

pytestmark = pytest.mark.gpu


def Call(*a, **k):
    return Both(*a, prefill=True, **k)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("t", (F32, F16, BF16))
@pytest.mark.parametrize("tiled", (False, True))
def test_heads(dev, heads, t, tiled):
    Call(dev, 1100, (70,) if heads[1] > 8 else (70, 3), *heads, tiled, t).upload().launch().check()


@pytest.mark.parametrize("m", (1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200))
@pytest.mark.parametrize("dk", (64, 128))
def test_lengths(dev, m, dk):
    Call(dev, 1110 + m, (m, m), 1, 2, dk, 32, ragged=False).upload().launch().check()


@pytest.mark.parametrize("new", [(1, 64, 63, 65), (0, 5, 0, 0, 130, 0), (64, 64), (3,) * 40, (100, 1, 28, 2, 190), (0, 0)])
@pytest.mark.parametrize("t", (F32, BF16))
def test_packed(dev, new, t):
    Call(dev, 1120, new, 2, 4, 64, 48, t=t, ragged=True, room=9).upload().launch().check()


@pytest.mark.parametrize("pad,ypad,t", [(0, 1, F32), (4, 4, F32), (3, 2, F32), (1, 0, F16), (4, 3, BF16), (2, 4, F16)])
def test_strides(dev, pad, ypad, t):
    Call(dev, 1130, (30, 90), 1, 2, 64, 48, False, t, pad=pad, ypad=ypad).upload().launch().check()


def test_slots(dev):
    """In place; from one slot, and from none; into no slot."""
    Call(dev, 1140, (66, 3), start=(1, 0), to=(1, 0)).upload().launch().check()
    Call(dev, 1141, (66, 66, 1, 70, 5), start=(6, 6, -1, 6, -1), to=(0, 1, 2, -1, -1)).upload().launch().check()


@pytest.mark.parametrize("keep", (0.99999, 0.9, 0.5, 1e-3, 1e-20))
@pytest.mark.parametrize("dk", (64, 128))
def test_decays(dev, keep, dk):
    Call(dev, 1150, (130, 70), 1, 2, dk, 32, keep=keep).upload().launch().check()


def test_scale_and_eps(dev):
    Call(dev, 1151, (70, 70), eps=0.5, scale=-3.0).upload().launch().check()


@pytest.mark.parametrize("amp", (1e-20, 1e-3, 1e4, 1e20))
def test_state_sizes(dev, amp):
    """States of other sizes than the values: columns of different sizes side by side."""
    c = Call(dev, 1152, (70, 9), 1, 2, 128, 48, amp=amp)
    c.S[..., ::5] *= np.float32(1e-8)
    c.S[..., 3::7] = 0
    c.upload().launch().check()


def test_value_sizes(dev):
    """Values of very different sizes in a chunk's columns and rows."""
    c = Call(dev, 1153, (130,), 1, 2, 64, 64)
    v = c.L.raw[:, 128:256]
    v *= (10.0 ** c.s.g.integers(-6, 7, (1, 128))).astype(np.float32)
    v[70:90] *= np.float32(1e-5)
    v[:, 9] = 0
    c.L.x = c.L.raw.astype(np.float64)
    c.upload().launch().check()


def test_extreme_gates(dev):
    c = Call(dev, 1154, (80, 80), 2, 4, 64, 32)
    c.L.ab[::3, :4] = np.float32([40, -40, 100, -100])
    c.L.ab[1::7, 4:8] = np.float32([200, -200, 88, -90])
    c.L.ab[5, :4] = 1e30
    c.L.A[:2] = 0, 3
    c.upload().launch().check()


@pytest.mark.parametrize("dk", (64, 128))
@pytest.mark.parametrize("keep", (0.99999, 0.9))
def test_like_keys(dev, dk, keep):
    """Keys that are all the same, or of two directions, with rates of almost 1: the system of a chunk is as far from diagonal as it gets."""
    c = Call(dev, 1155, (130, 130), 1, 2, dk, 32, keep=keep)
    k = c.L.raw[:, dk:2 * dk]
    k[:130] = k[0]
    k[130::2], k[131::2] = k[130], k[131]
    c.L.x = c.L.raw.astype(np.float64)
    c.L.ab[:, 2:4] = 12
    c.upload().launch().check()


def test_zero_keys(dev):
    c = Call(dev, 1156, (70, 4))
    c.L.raw[3:69, :256] = 0
    c.L.x[3:69, :256] = 0
    c.upload().launch().check()


def test_decode_goes_on(dev):
    """A prompt, then its next tokens by either operator: within both bounds of each other."""
    n, more = 100, 3
    p = Call(dev, 1157, (n + more,), 2, 4, 128, 64, tiled=True).upload().launch()
    whole, _ = p.results()
    first = Call(dev, 1157, (n + more,), 2, 4, 128, 64, tiled=True).upload()
    first.s.T = n
    first.launch()
    d, s = first.dev, first.s
    s.dstart.upload(s.to)
    q, k, v, a, b = first.L.args()
    w = first.L.w * 4 * n
    first.dev.gdn_decode(first.L.gdn, s.slots, first.dS, q + w, k + w, v + w, a + 4 * n * 9, b + 4 * n * 9, first.dy.ptr + n * first.ys * 4, F32, more, *first.L.strides(), first.ys)
    got, _ = first.results()
    _, err, _, _ = p.L.run64(s.at(0), p.S[p.s.start[0]], chunk=64)
    assert (np.abs(got.astype(np.float64) - whole) <= 2 * err.reshape(n + more, -1) + 2 * U * np.abs(whole)).all()


def some_heads(L, heads):
    """The layer of some value heads of L alone, each with a key head of its own."""
    c = copy.copy(L)
    c.n_k = c.n_v = len(heads)
    hk = [h % L.n_k if L.tiled else h * L.n_k // L.n_v for h in heads]
    col = [np.arange(o + h * d, o + (h + 1) * d) for o, hs, d in ((0, hk, L.dk), (L.n_k * L.dk, hk, L.dk), (2 * L.n_k * L.dk, heads, L.dv)) for h in hs]
    c.x, c.ab = L.x[:, np.concatenate(col)], L.ab[:, list(heads) + [L.n_v + h for h in heads]]
    c.A, c.dt, c.tiled = L.A[list(heads)], L.dt[list(heads)], False
    return c


def test_sequences_over_launches(dev):
    """More chunk slots than a pair of launches takes: sequences that begin in one and go on in the next, over several, in place."""
    n_k, n_v, dk, dv = 32, 128, 128, 16
    per = n_k * 3 * 64 * 128 * 4 + n_v * 25600
    most = (512 << 20) // per + 1  # slots of a pair of launches
    new = [64 * (most - 2) + 5, 64 * 3, 7, 64 * (2 * most) + 1, 64, 64 * most, 10]
    c = Call(dev, 1158, new, n_k, n_v, dk, dv, tiled=True, t=BF16, start=(0, -1, 2, 3, 4, -1, 6), to=(0, 1, 2, 3, 4, 5, -1)).upload().launch()
    dev.kv_check()
    raw, pool = c.results()
    s, heads = c.s, [3, 100]
    pool = state_of(pool.reshape(s.n_slots, n_v, dv // 16, dk, 16)).astype(np.float64)
    assert np.array_equal(pool[6:], c.S[6:])  # the last one's starting slot too
    y, L = from16(raw, BF16).reshape(-1, n_v, dv)[:, heads], some_heads(c.L, heads)
    for b in range(s.n):
        want, err, st, es = L.run64(s.at(b), c.S[s.start[b]][heads] if s.start[b] >= 0 else np.zeros((2, dk, dv)), chunk=64)
        near(y[s.at(b)], want, err * (1 + ULP[BF16]) + ULP[BF16] * np.abs(want) + TINY[BF16], f"sequence {b}")
        if s.to[b] >= 0:
            near(pool[s.to[b]][heads], st[-1], es[-1], f"state {b}")


def test_not_finite(dev):
    """What is not finite reaches its own column (a value) or head, from the beginning of its chunk at the earliest; other sequences and the
    chunks before are whole."""
    c = Call(dev, 1159, (140, 60), 2, 2, 64, 32)
    q, k, v = 0, 128, 256
    x = c.L.raw
    x[100, v + 5] = np.nan
    x[70, k + 64 + 7] = np.inf
    x[150, q + 3] = np.nan
    c.L.x = x.astype(np.float64)
    c.upload().launch()
    raw, pool = c.results()
    nan = np.isnan(raw.reshape(200, 2, 32))
    assert nan[100:140, 0, 5].all() and nan[70:140, 1].all() and nan[150, 0].all()
    allowed = np.zeros_like(nan)
    allowed[64:140, 0, 5] = allowed[64:140, 1] = allowed[150, 0] = True
    assert not (nan & ~allowed).any()
    st = np.isnan(pool.reshape(c.s.n_slots, 2, 2, 64, 16))
    assert st[c.s.to[0], 1].all() and st[c.s.to[0], 0, 0, :, 5].all() and st.sum() == 2 * 64 * 16 + 64


def test_bad_slots(dev):
    c = Call(dev, 1160, (70, 3, 66), 1, 2, 64, 32)
    n = c.s.n_slots
    for start, to, lost in (((n, 1, 2), (3, 4, 5), 0), ((0, -2, 2), (3, 4, 5), 1), ((0, 1, 2), (3, 4, n), None), ((0, 1, 2), (-(1 << 31), 4, 5), None)):
        c.s.start, c.s.to = np.array(start, np.int32), np.array(to, np.int32)
        c.upload().launch()
        with pytest.raises(dev.AmdcError, match="slot outside"):
            dev.kv_check()
        dev.kv_check()
        raw, pool = c.results()
        if lost is not None:
            at = c.s.at(lost)
            assert np.isnan(raw[at]).all() and not np.isnan(np.delete(raw, range(at.start, at.stop), 0)).any()
            assert np.array_equal(pool.reshape(c.S.shape[0], -1)[to[lost]], pool_of(c.S)[to[lost]].ravel())
        else:
            c.s.to = np.where((c.s.to < 0) | (c.s.to >= n), -1, c.s.to)
            c.check()


@pytest.mark.parametrize("cu", [(0, 70, 60, 139), (-1, 70, 73, 139), (0, 70, 73, 150), (0, 1 << 30, 73, 139), (5, 5, 5, 5)])
def test_rows_out_of_bounds(dev, cu):
    """Of a sequence with rows outside 0 .. T none is written."""
    c = Call(dev, 1161, (70, 3, 66), 1, 2, 64, 32, room=4).upload()
    c.s.dcu.upload(np.array(cu, np.int32))
    c.launch()
    if cu == (5, 5, 5, 5):
        dev.kv_check()
    else:
        with pytest.raises(dev.AmdcError, match="rows outside"):
            dev.kv_check()
    dev.kv_check()
    raw, _ = c.results()
    good = np.zeros(len(raw), bool)
    for a, b in zip(cu, cu[1:]):
        if 0 <= a <= b <= c.s.T:
            good[a:b] = True
    assert (raw[~good] == 7).all()


def test_graph(dev):
    c = Call(dev, 1162, (64, 5, 80), 2, 4, 128, 64, True, BF16, room=7).upload()
    s = dev.Stream()
    graph = dev.Graph(s, lambda st: c.launch(st))
    new = list(c.s.new)
    for k in range(3):
        # the same rows dealt otherwise, other slots
        c.s.new = new[k:] + new[:k]
        c.s.cu = np.concatenate([[0], np.cumsum(c.s.new)]).astype(np.int32)
        c.s.start, c.s.to = np.roll(c.s.start, 1), np.roll(c.s.to, 1)
        c.s.dcu.upload(c.s.cu), c.s.dstart.upload(c.s.start), c.s.dto.upload(c.s.to)
        c.dS.upload(pool_of(c.S)), c.dy.upload(c.y0)
        graph.launch()
        s.sync()
        c.check()
    del graph


def test_same_bits(dev):
    c = Call(dev, 1163, (300, 77, 1), 2, 6, 128, 64, True, F32).upload().launch()
    y, p = c.results()
    for _ in range(3):
        c.dS.upload(pool_of(c.S)), c.ws.fill(0x7F)
        c.launch()
        y2, p2 = c.results()
        assert np.array_equal(y, y2) and np.array_equal(p, p2)


@pytest.mark.parametrize("t", (F32, BF16))
@pytest.mark.parametrize("new", [(1,) * 20 + (70, 16, 17, 1, 0, 200, 15), (16, 17), (130, 1), (1, 2, 3), (0, 0, 5)])
def test_mixed(dev, new, t):
    """Decode steps beside prompts: the sequences of a few rows go token after token, the others in chunks."""
    Call(dev, 1170, new, 2, 6, 128, 64, True, t, ragged=True, room=3).upload().launch().check()


def test_few_as_decode(dev):
    """T rows of every sequence, few of them: decode's bits, packed or not."""
    d = Both(dev, 1171, (5,) * 9, 2, 4, 64, 48).upload().launch()
    y, p = d.results()
    for ragged in (False, True):
        c = Call(dev, 1171, (5,) * 9, 2, 4, 64, 48, ragged=ragged).upload().launch()
        y2, p2 = c.results()
        assert np.array_equal(y, y2) and np.array_equal(p, p2)
