"""amdc_conv against the definition in 64 bits: one token, verify steps with a state kept after each, packed prompts; odd numbers of
channels, widths, strides and lengths around the units that the rows are dealt in; states in place."""
import numpy as np
import pytest

from attncase import BF16, F16, F32, TINY, ULP, as_float
from lincase import NAN, U, Seqs, conv64, near

pytestmark = pytest.mark.gpu


class Call:
    def __init__(self, dev, seed, new, ch, width=4, t=F32, act=1, bias=True, xpad=0, ypad=0, **kw):
        s = self.s = Seqs(dev, seed, new, **kw)
        g, self.dev, self.ch, self.width, self.t, self.act = s.g, dev, ch, width, t, act
        self.x = g.standard_normal((s.total, ch + xpad)).astype(np.float32)
        self.x[s.rows:] = NAN
        if xpad:
            self.x[:, ch:] = NAN
        self.w = (g.standard_normal((ch, width)) / 2).astype(np.float32)
        self.bias = g.standard_normal(ch).astype(np.float32) if bias else None
        self.pool = g.standard_normal((s.n_slots, width - 1, ch)).astype(np.float32)
        self.xs, self.ys = ch + xpad, ch + ypad
        self.y0 = np.full((s.total, self.ys), 7, np.float32 if t == F32 else np.uint16)

    def upload(self):
        d = self.dev
        self.s.upload()
        self.dx, self.dw, self.db = d.DevBuf.of(self.x), d.DevBuf.of(self.w), None if self.bias is None else d.DevBuf.of(self.bias)
        self.dpool, self.dy = d.DevBuf.of(self.pool), d.DevBuf.of(self.y0)
        return self

    def launch(self, stream=None):
        s = self.s
        self.dev.conv(s.slots, self.dpool, self.dx, self.dw, self.db, self.dy, self.t, self.ch, self.width, s.T, self.xs, self.ys, cu=s.dcu if s.ragged else None, each=s.each,
                      act=self.act, stream=stream)
        return self

    def check(self, bad=()):
        """bad: sequences whose rows are NaN and whose slots stay."""
        s = self.s
        raw = self.dy.download(self.y0.dtype).reshape(self.y0.shape)
        y = as_float(raw, self.t)[:, :self.ch]
        states = []
        for b in range(s.n):
            old = self.pool[s.start[b]] if s.start[b] >= 0 else np.zeros_like(self.pool[0])
            want, mag, pre, st = conv64(self.x[s.at(b)][:, :self.ch], self.w, self.bias, old, self.act)
            # a rounding a term; SiLU multiplies by sigmoid(v), whose slope times v is at most 1.1 of it, and whose exp2 and
            # reciprocal are off by (3 + |v|) u each way
            err = U * (self.width + 1) * mag * (1.2 if self.act else 1) + (U * (6 + 2 * np.abs(pre)) * np.abs(want) if self.act else 0)
            near(y[s.at(b)], want, err * (1 + ULP[self.t]) + ULP[self.t] * np.abs(want) + TINY[self.t], f"sequence {b}")
            states.append(st)
        assert np.array_equal(self.dpool.download(np.float32).reshape(self.pool.shape), s.after(self.pool, states).astype(np.float32))
        assert (raw[s.rows:] == 7).all() and (raw[:, self.ch:] == 7).all()


@pytest.mark.parametrize("ch,width,t", [(10240, 4, F32), (8192, 4, BF16), (64, 2, F16), (1, 4, F32), (3, 3, F32), (257, 4, F16), (1026, 3, BF16), (6, 2, F32)])
@pytest.mark.parametrize("new", [(1,), (1, 1, 1), (5, 5)])
def test_decode(dev, ch, width, t, new):
    Call(dev, 900 + ch, new, ch, width, t).upload().launch().check()


@pytest.mark.parametrize("ch,width,t", [(640, 4, F32), (1028, 4, BF16), (77, 3, F16), (96, 2, F32)])
@pytest.mark.parametrize("new", [(1, 2, 3, 4), (31, 32, 33), (64, 1, 65), (0, 7, 0, 100), (300,), (8, 9, 40, 41)])
def test_packed(dev, ch, width, t, new):
    Call(dev, 910 + ch, new, ch, width, t, ragged=True, room=5).upload().launch().check()


@pytest.mark.parametrize("t", (F32, F16))
@pytest.mark.parametrize("T", (1, 2, 3, 5, 16))
@pytest.mark.parametrize("width", (2, 3, 4))
def test_verify(dev, width, t, T):
    """The state after every token, the last one in the slot that the sequence started from."""
    s = Seqs(dev, 920, (T, T, T), each=True)
    to = s.to.copy()
    to[[T - 1, 2 * T - 1]] = s.start[:2]
    Call(dev, 920, (T, T, T), 132, width, t, each=True, start=s.start, to=to).upload().launch().check()


@pytest.mark.parametrize("new", [(1, 1), (2, 2), (3, 3), (70, 70), (2, 50, 1, 33)])
def test_in_place(dev, new):
    n = len(new)
    Call(dev, 930, new, 300, start=np.arange(n)[::-1], to=np.arange(n)[::-1]).upload().launch().check()


def test_no_slots(dev):
    """From zeros, and the new state nowhere."""
    Call(dev, 931, (5, 9, 40), 68, start=(-1, 3, -1), to=(0, -1, -1)).upload().launch().check()


@pytest.mark.parametrize("xpad,ypad,t", [(4, 0, F32), (1, 0, F32), (0, 1, F16), (0, 2, BF16), (3, 5, F32), (8, 4, BF16)])
def test_strides(dev, xpad, ypad, t):
    Call(dev, 940, (3, 34), 132, t=t, xpad=xpad, ypad=ypad, bias=False).upload().launch().check()


def test_no_act(dev):
    Call(dev, 941, (2, 34), 132, act=0).upload().launch().check()


def test_far_values(dev):
    """Outputs where exp(-v) overflows or vanishes."""
    c = Call(dev, 942, (40,), 16)
    c.x *= 300
    c.upload().launch().check()


def test_many_sequences(dev):
    new = [int(v) for v in np.random.default_rng(5).integers(0, 40, 700)]
    Call(dev, 943, new, 40).upload().launch().check()


def test_bad_slots(dev):
    """A sequence from outside the pool: NaN rows, no state written; a slot to outside it: not written. The others are whole."""
    c = Call(dev, 944, (3, 40, 5), 36)
    n = c.s.n_slots
    for start, to, lost in (((n, 1, 2), (3, 4, 5), 0), ((0, -2, 2), (3, 4, 5), 1), ((0, 1, 2), (3, 4, n), None), ((0, 1, 2), (3, -7, 5), None)):
        c.s.start, c.s.to = np.array(start, np.int32), np.array(to, np.int32)
        c.upload().launch()
        with pytest.raises(dev.AmdcError, match="slot outside"):
            dev.kv_check()
        dev.kv_check()
        s = c.s
        if lost is not None:
            y = c.dy.download(np.float32).reshape(c.y0.shape)
            assert np.isnan(y[s.at(lost)][0]).all()  # the whole window of its first row
            pool = c.dpool.download(np.float32).reshape(c.pool.shape)
            assert np.array_equal(pool[to[lost]], c.pool[to[lost]])
        else:
            s.to = np.where((s.to < 0) | (s.to >= n), -1, s.to)
            c.check()


def test_bad_rows(dev):
    c = Call(dev, 945, (3, 40, 5), 36, room=3)
    for cu in ((0, 3, 2, 48), (-1, 3, 43, 48), (0, 3, 43, 52)):
        c.upload()
        c.s.dcu.upload(np.array(cu, np.int32))
        c.launch()
        with pytest.raises(dev.AmdcError, match="rows outside"):
            dev.kv_check()
        dev.kv_check()


def test_graph(dev):
    """Captured once; the host moves slots and rows on between replays."""
    c = Call(dev, 946, (4, 30), 260, room=6).upload()
    s = dev.Stream()
    graph = dev.Graph(s, lambda st: c.launch(st))
    for k in range(3):
        c.s.start, c.s.to = np.roll(c.s.start, 1), np.roll(c.s.to, 1)
        c.s.dstart.upload(c.s.start), c.s.dto.upload(c.s.to)
        c.dpool.upload(c.pool), c.dy.upload(c.y0)
        graph.launch()
        s.sync()
        c.check()
    del graph
