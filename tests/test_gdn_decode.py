"""amdc_gdn_decode against the recurrence in 64 bits: one and a few tokens, all head sizes and both orders of heads, the three
types, strides; states in place, shared to start from, and kept after every token."""
import numpy as np
import pytest

from attncase import BF16, F16, F32, TINY, ULP, as_float
from lincase import Layer, Seqs, near, pool_of, state_of

pytestmark = pytest.mark.gpu


class Call:
    """Also of amdc_gdn_prefill (chunk: the tokens that it takes together)."""

    def __init__(self, dev, seed, new, n_k=2, n_v=4, dk=64, dv=64, tiled=False, t=F32, pad=0, ypad=0, amp=0.3, prefill=False, keep=None, eps=1e-6, scale=None, **kw):
        s = self.s = Seqs(dev, seed, new, **kw)
        self.dev, self.t, self.prefill = dev, t, prefill
        self.L = Layer(s.g, s.rows, n_k, n_v, dk, dv, tiled, t, eps=eps, scale=scale, pad=pad, room=s.total - s.rows, keep=keep)
        self.S = (amp * s.g.standard_normal((s.n_slots, n_v, dk, dv))).astype(np.float32)
        self.ys = n_v * dv + ypad
        self.y0 = np.full((s.total, self.ys), 7, np.float32 if t == F32 else np.uint16)

    def upload(self):
        self.s.upload()
        self.L.upload(self.dev)
        self.dS, self.dy = self.dev.DevBuf.of(pool_of(self.S)), self.dev.DevBuf.of(self.y0)
        if self.prefill:
            self.ws = self.dev.DevBuf(self.dev.gdn_prefill_ws(self.L.gdn, self.s.n, self.s.total if self.s.ragged else self.s.n * self.s.T))
            self.ws.fill(0xFF)  # of any content
        return self

    def launch(self, stream=None):
        s, d, L = self.s, self.dev, self.L
        if self.prefill:
            d.gdn_prefill(L.gdn, s.slots, self.dS, *L.args(), self.dy, self.t, s.T, *L.strides(), self.ys, self.ws, self.ws.nbytes, cu=s.dcu if s.ragged else None, stream=stream)
        else:
            d.gdn_decode(L.gdn, s.slots, self.dS, *L.args(), self.dy, self.t, s.T, *L.strides(), self.ys, each=s.each, stream=stream)
        return self

    def results(self):
        raw = self.dy.download(self.y0.dtype).reshape(self.y0.shape)
        return raw, self.dS.download(np.float32)

    def check(self):
        s, L = self.s, self.L
        raw, pool = self.results()
        w = L.n_v * L.dv
        y = as_float(raw, self.t)[:, :w].reshape(-1, L.n_v, L.dv)
        states, errs = [], []
        for b in range(s.n):
            old = self.S[s.start[b]] if s.start[b] >= 0 else np.zeros_like(self.S[0])
            want, err, st, es = L.run64(s.at(b), old, chunk=64 if self.prefill else 1)
            near(y[s.at(b)], want, err * (1 + ULP[self.t]) + ULP[self.t] * np.abs(want) + TINY[self.t], f"sequence {b}")
            states.append(st), errs.append(es)
        near(state_of(pool.reshape(s.n_slots, L.n_v, L.dv // 16, L.dk, 16)).astype(np.float64), s.after(self.S.astype(np.float64), states),
             s.after(np.zeros(self.S.shape), errs), "states")
        assert (raw[s.rows:] == 7).all() and (raw[:, w:] == 7).all()
        return self


HEADS = [(2, 4, 64, 64), (1, 1, 128, 128), (16, 48, 128, 128), (2, 6, 128, 64), (3, 3, 64, 128), (1, 5, 64, 16), (2, 2, 128, 48), (1, 2, 64, 256)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("t", (F32, F16, BF16))
@pytest.mark.parametrize("tiled", (False, True))
def test_one_token(dev, heads, t, tiled):
    Call(dev, 1000, (1,) * (1 if heads[1] > 8 else 3), *heads, tiled, t).upload().launch().check()


@pytest.mark.parametrize("T", (2, 3, 5, 16))
@pytest.mark.parametrize("each", (False, True))
@pytest.mark.parametrize("t", (F32, BF16))
def test_few_tokens(dev, T, each, t):
    Call(dev, 1010 + T, (T, T), 2, 6, 128, 32, True, t, each=each).upload().launch().check()


@pytest.mark.parametrize("pad,ypad,t", [(0, 1, F32), (4, 4, F32), (3, 2, F32), (1, 0, F16), (4, 3, BF16), (2, 4, F16)])
def test_strides(dev, pad, ypad, t):
    Call(dev, 1020, (3, 3), 1, 2, 64, 48, False, t, pad=pad, ypad=ypad).upload().launch().check()


def test_in_place(dev):
    Call(dev, 1030, (1,) * 5, start=(4, 0, 2, 1, 3), to=(4, 0, 2, 1, 3)).upload().launch().check()
    # a verify step whose last state goes back to where it came from
    Call(dev, 1031, (3, 3), each=True, start=(0, 1), to=(2, 3, 0, 4, 5, 1)).upload().launch().check()


def test_shared_start(dev):
    """Several sequences that start from one slot, and from none."""
    Call(dev, 1032, (2,) * 5, start=(6, 6, -1, 6, -1), to=(0, 1, 2, -1, -1)).upload().launch().check()


@pytest.mark.parametrize("keep", (0.9999, 0.5, 1e-3))
def test_decays(dev, keep):
    Call(dev, 1040, (16, 16), 1, 2, 128, 32, keep=keep).upload().launch().check()


def test_scale_and_eps(dev):
    Call(dev, 1041, (2, 2), eps=0.5, scale=-3.0).upload().launch().check()


def test_extreme_gates(dev):
    """Gates at the ends of their ranges: softplus and the sigmoids far out, a decay that underflows, an A of 0 and one above it."""
    c = Call(dev, 1042, (8, 8), 2, 4, 64, 32)
    c.L.ab[:, :8] = np.float32([0, 40, -40, 100, -100, 1e4, -1e4, 3])
    c.L.ab[8:, :8] = np.float32([-200, 90, 20, -20, 88, -88, 0.5, 1e30])
    c.L.A[:2] = 0, 3
    c.upload().launch().check()


def test_zero_keys(dev):
    """A key or query of zeros is one of norm 0: the state only decays."""
    c = Call(dev, 1043, (4, 4))
    c.L.raw[1:3, :256] = 0
    c.L.x[1:3, :256] = 0
    c.upload().launch().check()


def test_sixteen_hundred_sequences(dev):
    Call(dev, 1044, (1,) * 1600, 1, 2, 64, 16).upload().launch().check()


def test_not_finite(dev):
    """A value that is not finite stays in its column, a key in its head, a query in its row, and none goes back in time."""
    c = Call(dev, 1045, (6, 6), 2, 2, 64, 32)
    q, k, v = 0, 128, 256
    x = c.L.raw
    x[2, v + 5] = np.nan          # head 0, column 5, from row 2 on
    x[3, k + 64 + 7] = np.inf     # head 1, from row 3 on
    x[7, q + 3] = np.nan          # sequence 1, row 1, head 0
    c.L.x = x.astype(np.float64)
    c.upload().launch()
    raw, _ = c.results()
    y = raw.reshape(12, 2, 32)
    nan = np.isnan(y)
    want = np.zeros_like(nan)
    want[2:6, 0, 5] = want[3:6, 1] = want[7, 0] = True
    assert np.array_equal(nan, want)


def test_bad_slots(dev):
    c = Call(dev, 1046, (2, 2, 2), 1, 2, 64, 32)
    n = c.s.n_slots
    for start, to, lost in (((n, 1, 2), (3, 4, 5), 0), ((0, -2, 2), (3, 4, 5), 1), ((0, 1, 2), (3, 4, n), None), ((0, 1, 2), (3, -(1 << 31), 5), None)):
        c.s.start, c.s.to = np.array(start, np.int32), np.array(to, np.int32)
        c.upload().launch()
        with pytest.raises(dev.AmdcError, match="slot outside"):
            dev.kv_check()
        dev.kv_check()
        raw, pool = c.results()
        if lost is not None:
            assert np.isnan(raw[c.s.at(lost)]).all() and not np.isnan(np.delete(raw, range(2 * lost, 2 * lost + 2), 0)).any()
            assert np.array_equal(pool.reshape(c.S.shape[0], -1)[to[lost]], pool_of(c.S)[to[lost]].ravel())
        else:
            c.s.to = np.where((c.s.to < 0) | (c.s.to >= n), -1, c.s.to)
            c.check()


def test_graph(dev):
    c = Call(dev, 1047, (1, 1, 1), 2, 4, 128, 64, True, BF16).upload()
    s = dev.Stream()
    graph = dev.Graph(s, lambda st: c.launch(st))
    for k in range(3):
        c.s.start, c.s.to = np.roll(c.s.start, 1), np.roll(c.s.to, 1)
        c.s.dstart.upload(c.s.start), c.s.dto.upload(c.s.to)
        c.dS.upload(pool_of(c.S)), c.dy.upload(c.y0)
        graph.launch()
        s.sync()
        c.check()
    del graph


def test_far_slots(dev):
    """Slots behind 2^32 values of the pool."""
    n_v, dk, dv = 16, 128, 128
    per = n_v * dk * dv
    n = (1 << 32) // per + 3
    c = Call(dev, 1048, (1, 1), 4, n_v, dk, dv)
    s = c.s
    pool = dev.DevBuf(4 * per * n)
    c.upload()
    mine = pool_of(c.S).reshape(s.n_slots, per)
    for i in range(2):
        pool.upload(mine[s.start[i]], 4 * per * (n - 1 - i))
    s.dstart.upload(np.array([n - 1, n - 2], np.int32)), s.dto.upload(np.array([n - 3, n - 1], np.int32))
    dev.gdn_decode(c.L.gdn, dev.Slots(2, n, s.dstart, s.dto), pool, *c.L.args(), c.dy, F32, 1, *c.L.strides(), c.ys)
    dev.kv_check()
    for i, at in enumerate((n - 3, n - 1)):
        c.dS.upload(pool.download(np.float32, per, 4 * per * at), 4 * per * int(s.to[i]))
    c.check()
