"""amdc_attn_decode against the definition in 64 bits on the cache's stored values. Positions that a row does not see hold NaN
unless a test says otherwise (attncase.Case fills the pools with it)."""
import numpy as np
import pytest

from attncase import BF16, F16, F32, TINY, ULP, Case, as_float, attn64, to16

pytestmark = pytest.mark.gpu


def bound(c, t, y, av, aq, L):
    """How far an output may be off: a weight is off by a factor of 1 + e at most, with e the sum of
    - its own rounding (16-bit: half a step; f32: two f16 or three bf16 parts, 2^-22, and the exponential's 2^-22),
    - the score's error: the query's parts (2^-22), and one rounding to each of hd products' sums in every part,
    - a rounding of the sum at each of L / 32 steps and some 64 joins and rescalings;
    it enters the sum of weighted values and the sum of weights, hence twice; then the result's own rounding."""
    parts = {F32: 2 if c.type == F16 else 3}.get(t, 1)
    e = (2.0 ** -21 if t == F32 else ULP[t] + 2.0 ** -22) + aq[:, :, None] * (2.0 ** -22 + parts * (c.hd + 8) * 2.0 ** -24) + (L / 32 + 64) * 2.0 ** -24
    return 2 * e * av + ULP[t] * np.abs(y) * (1 + 2 * e) + TINY[t]


class Call:
    def __init__(self, c, t, T, window=0, scale=None, pad=0, off=0, q=None, q8=False, y=True, amp=2.0):
        dev, self.c, self.t, self.T, self.window = c.dev, c, t, T, window
        w = c.n_q * c.hd
        self.scale = np.float32(1 / np.sqrt(c.hd) if scale is None else scale)
        self.qs, self.ys, self.off = w + pad, w + 2 * pad, off
        rows = c.n_seq * T
        q = (amp * c.g.standard_normal((rows, w))).astype(np.float32) if q is None else q.reshape(rows, w).astype(np.float32)
        buf = np.zeros(off + rows * self.qs, np.float32)
        buf[off:].reshape(rows, self.qs)[:, :w] = q
        raw = buf if t == F32 else to16(buf, t)
        self.q = as_float(raw, t)[off:].reshape(rows, self.qs)[:, :w].reshape(rows, c.n_q, c.hd)
        esz = self.esz = 4 if t == F32 else 2
        self.Q, self.Y = dev.DevBuf.of(raw), dev.DevBuf((off + rows * self.ys) * esz) if y else None
        if y:
            self.Y.fill(0x5A)
        self.q8s = w // 32 * 40 + 4 * pad
        self.Q8 = dev.DevBuf(rows * self.q8s) if q8 else None
        if q8:
            self.Q8.fill(0xA5)
        self.size = dev.attn_decode_ws(c.kv, c.n_q, T)
        self.ws = dev.DevBuf(self.size)
        self.ws.fill(0)
        self.rows, self.w = rows, w

    def launch(self, stream=None, ws=None):
        c = self.c
        c.dev.attn_decode(c.kv, self.Q.ptr + self.off * self.esz, self.Y.ptr + self.off * self.esz if self.Y else None, self.t, c.n_q, self.T, self.qs, self.ys, self.scale,
                          (ws or self.ws), (ws or self.ws).nbytes, window=self.window, q8=self.Q8, q8s=self.q8s if self.Q8 else 0, stream=stream)
        return self

    def got(self):
        self.c.dev.sync()
        raw = self.Y.download(np.float32 if self.t == F32 else np.uint16)
        rows = raw[self.off:].reshape(self.rows, self.ys)
        untouched = np.concatenate([raw[:self.off].ravel(), rows[:, self.w:].ravel()])
        assert np.all(untouched.view(np.uint8) == 0x5A), "something beside the rows was written"
        return as_float(rows[:, :self.w].copy(), self.t).reshape(self.rows, self.c.n_q, self.c.hd)

    def check(self, lens=None):
        c, T = self.c, self.T
        y = self.got()
        lens = c.lens if lens is None else lens
        for b, L in enumerate(lens):
            mine = y[b * T:(b + 1) * T]
            if L == 0:
                assert np.all(mine == 0), f"sequence {b} of no positions"
                continue
            k, v = c.stored(b)
            want, av, aq = attn64(self.q[b * T:(b + 1) * T], k, v, float(self.scale), np.arange(L - T, L), self.window)
            off = np.abs(mine - want) / bound(c, self.t, want, av, aq, L)
            assert off.max() <= 1, f"sequence {b} of {L}: {off.max():.2f} of the bound at {np.unravel_index(off.argmax(), off.shape)}, {int((~(off <= 1)).sum())} values"
            assert not np.isnan(off).any()
        counters = self.ws.download(np.uint32, 16384)
        assert not counters.any(), "a counter was left"
        c.dev.kv_check()
        return y


CASES = [
    # type, t, n_q, n_kv, hd, page, T, window, lens
    (F16, F32, 4, 4, 128, 16, 1, 0, (1,)),
    (F16, F16, 4, 2, 64, 16, 1, 0, (1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 127, 129)),
    (F16, F32, 32, 32, 128, 64, 1, 0, (421,)),
    (F16, F32, 24, 4, 256, 64, 1, 0, (5000,)),  # split over the length
    (BF16, BF16, 8, 1, 256, 32, 1, 0, (20011,)),  # two levels of joins
    (BF16, F32, 8, 2, 128, 128, 1, 0, (3000, 17, 999)),
    (F16, F32, 16, 1, 64, 16, 1, 0, (9000, 1, 0, 4001)),
    (BF16, F32, 6, 3, 64, 32, 1, 100, (40, 100, 101, 350, 1000)),
    (F16, F16, 8, 2, 128, 16, 1, 1, (5, 64, 33)),  # a window of the row itself
    (F16, F32, 24, 4, 256, 64, 5, 0, (300, 5, 64, 2000)),  # 30 columns: two blocks
    (BF16, BF16, 32, 8, 128, 16, 8, 0, (100, 8, 1500)),  # 32 columns
    (F16, F16, 5, 1, 64, 32, 3, 7, (4, 33, 200)),  # 15 columns; a window inside the new rows
    (F16, F32, 128, 1, 64, 16, 1, 0, (77, 1000)),  # 8 blocks of columns
    (BF16, F32, 14, 2, 256, 16, 4, 300, (301, 700)),
    (F16, F16, 12, 12, 64, 16, 16, 0, (16, 17, 90)),
    (BF16, BF16, 8, 8, 128, 16, 1, 0, tuple(20 + 37 * i % 400 for i in range(150))),  # over 128 sequences
    (F16, F16, 4, 1, 128, 16, 1, 0, tuple(1 + (i * i * 7) % 3000 for i in range(70))),
    (F16, F32, 2, 1, 128, 64, 1, 0, (190_000,)),  # chunks long enough for nontemporal loads
    (BF16, BF16, 6, 1, 256, 16, 1, 0, (90_000, 33_000)),
    (F16, F16, 32, 1, 128, 16, 1, 0, (5000, 1, 300)),  # one block of 32 columns, split
    (BF16, F32, 20, 1, 64, 16, 3, 0, (3000, 70)),  # blocks of 32 and 28
    (F16, F16, 128, 128, 64, 16, 1, 0, (700, 31)),  # more heads than CUs leave room for
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_decode(dev, i):
    ty, t, n_q, n_kv, hd, page, T, window, lens = CASES[i]
    print(CASES[i] if len(lens) < 20 else CASES[i][:-1], flush=True)
    c = Case(dev, 200 + i, ty, n_q, n_kv, hd, page, lens, (T,) * len(lens)).fill_all().upload()
    Call(c, t, T, window).launch().check()


@pytest.mark.parametrize("t", (F32, F16))
def test_rows_that_are_not_aligned(dev, t):
    c = Case(dev, 1, F16, 4, 2, 128, 16, (70, 300), (2, 2)).fill_all().upload()
    Call(c, t, 2, pad=3, off=1).launch().check()


def test_q8_copy(dev, orc):
    """The Q8 copy is amdc_quant_q8's of the f32 result, with y, without it, and beside a 16-bit y."""
    for n, (t, hd, lens) in enumerate(((F32, 64, (40, 0, 3000)), (F32, 128, (9, 800)), (F32, 256, (500, 77)))):
        c = Case(dev, 20 + n, F16, 8, 2, hd, 16, lens, (2,) * len(lens)).fill_all().upload()
        a = Call(c, t, 2, q8=True, pad=1)
        y = a.launch().check().astype(np.float32).reshape(a.rows, a.w)
        want = orc.quant_q8(y)
        got = a.Q8.download(np.uint8).reshape(a.rows, a.q8s)
        assert np.array_equal(got[:, :want.shape[1]], want)
        assert np.all(got[:, want.shape[1]:] == 0xA5)
        a.Q8.fill(0)
        a.Y = None
        a.launch()
        dev.sync()
        assert np.array_equal(a.Q8.download(np.uint8).reshape(a.rows, a.q8s)[:, :want.shape[1]], want)
    # a 16-bit y: the copy is of the values before y's rounding, a step of y off at most
    c = Case(dev, 29, BF16, 8, 2, 128, 16, (100, 5), (1, 1)).fill_all().upload()
    a = Call(c, BF16, 1, q8=True)
    y = a.launch().check().reshape(a.rows, a.w // 32, 32)
    q = a.Q8.download(np.uint8).reshape(a.rows, a.q8s)
    nb = a.w // 32
    d = q[:, 32 * nb:36 * nb].copy().view(np.float32).astype(np.float64)
    back = q[:, :32 * nb].copy().view(np.int8).astype(np.float64).reshape(a.rows, nb, 32) * d[:, :, None]
    assert (np.abs(back - y) <= d[:, :, None] * (0.5 + 2.0 ** -14) + ULP[BF16] * np.abs(y) * (1 + 2.0 ** -7)).all()


def test_infinities_where_rows_do_not_see(dev):
    """Three new tokens, the second's and third's values infinite or NaN, keys too: the earlier rows' results are as if they were not
    there; the rows that see an infinite value are infinite (f32: or NaN) in that value alone."""
    for ty, t in ((F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)):
        c = Case(dev, 31, ty, 6, 2, 128, 16, (45, 130), (3, 3)).fill_all()
        for b, L in enumerate(c.lens):
            k, v = c.k[b].copy(), c.v[b].copy()
            v[L - 2, :, 5], v[L - 1, :, 7], k[L - 1, :, 3] = np.inf, np.nan, np.nan
            c.put(b, L - 2, L, k, v)
        c.upload()
        y = Call(c, t, 3).launch()
        got = y.got()
        for b, L in enumerate(c.lens):
            k, v = c.stored(b)
            q = y.q[3 * b:3 * b + 3]
            want, av, aq = attn64(q[:1], k, v, float(y.scale), [L - 3], 0)
            assert (np.abs(got[3 * b:3 * b + 1] - want) <= bound(c, t, want, av, aq, L)).all()
            mid = got[3 * b + 1]
            # in f32 a weight goes in as p = p1 + p2 (+ p3), and p2 may be 0 or negative: p1 inf + p2 inf is inf or NaN
            assert (mid[:, 5] == np.inf).all() if t != F32 else (~np.isfinite(mid[:, 5])).all()
            v2 = np.where(np.isfinite(v), v, 0.0)
            want, av, aq = attn64(q[1:2], k, v2, float(y.scale), [L - 2], 0)
            keep = np.arange(128) != 5
            assert (np.abs(mid - want[0]) <= bound(c, t, want, av, aq, L)[0])[:, keep].all()
            assert np.isnan(got[3 * b + 2]).all()  # its own key is NaN


def test_infinities_before_the_window(dev):
    c = Case(dev, 33, F16, 4, 2, 64, 16, (300, 90), (2, 2)).fill_all()
    for b, L in enumerate(c.lens):
        v = np.full_like(c.v[b], np.nan)
        c.put(b, 0, L - 2 + 1 - 40, np.full_like(c.k[b], np.inf), v)  # the first row sees 40 positions back
    c.upload()
    Call(c, F32, 2, window=40).launch().check()
    Call(c, F16, 2, window=40).launch().check()


@pytest.mark.parametrize("ty,hd,page", [(F16, 64, 16), (BF16, 128, 16), (F16, 128, 32), (F16, 256, 16)])
def test_pages_before_the_window(dev, ty, hd, page):
    """Entries of pages that are wholly before every row's window, given back to the pool, may be anything."""
    lens, T, window = (300, 77, 90, 2000), 2, 40
    c = Case(dev, 60, ty, 8, 2, hd, page, lens, (T,) * 4).fill_all().upload()
    gone = c.table.copy()
    for b, L in enumerate(lens):
        gone[b, :max(0, L - T + 1 - window) // page] = (-1, 999999, 0x7FFFFFFF, -2 ** 31)[b]
    c.dtable.upload(gone)
    for t in (F32, ty):
        Call(c, t, T, window=window).launch().check()
    dev.kv_check()


def test_extreme_scores(dev):
    """Queries over f16's range (scaled down again by the scale), tiny ones, rows of zero, scores hundreds apart, a negative scale."""
    c = Case(dev, 35, F16, 4, 2, 128, 16, (200, 33), (1, 1)).fill_all().upload()
    q = c.g.standard_normal((2, 4 * 128))
    Call(c, F32, 1, q=q * 1e9, scale=1e-9 / 11).launch().check()
    Call(c, F32, 1, q=q * 1e-30, scale=1e30 / 11).launch().check()
    Call(c, F32, 1, q=q * 0).launch().check()
    Call(c, F32, 1, q=q * 40).launch().check()
    Call(c, F16, 1, q=q * 40).launch().check()
    Call(c, F32, 1, q=q, scale=-0.3).launch().check()
    Call(c, F32, 1, q=q, scale=0.0).launch().check()
    c = Case(dev, 36, BF16, 4, 2, 64, 16, (200, 33), (1, 1), amp=1e15).fill_all().upload()
    q = c.g.standard_normal((2, 4 * 64))
    Call(c, F32, 1, q=q * 1e15, scale=1e-30).launch().check()
    Call(c, BF16, 1, q=q * 1e15, scale=1e-30).launch().check()


def test_scales_of_zero_and_near_it(dev):
    """Scale 0 is the mean, whatever the products; a subnormal scale of products near f32's largest."""
    c = Case(dev, 61, BF16, 4, 2, 64, 16, (100, 33), (1, 1), amp=1e18).fill_all().upload()
    q = c.g.standard_normal((2, 4 * 64))
    for t in (F32, BF16):
        Call(c, t, 1, q=q * 1e18, scale=0.0).launch().check()
        Call(c, t, 1, q=q * 1e18, scale=1e-39).launch().check()


def test_rising_scores(dev):
    """Scores that grow along the sequence: the maximum is raised again and again."""
    c = Case(dev, 37, F16, 2, 2, 64, 16, (2500,), (1,))
    q = np.ones((1, 2 * 64))
    c.k[0][:] = (np.arange(2500) / 400 - 3)[:, None, None] + 0.01 * c.k[0]
    c.fill_all().upload()
    for t in (F32, F16):
        Call(c, t, 1, q=q, scale=0.5).launch().check()
    c.k[0][:] = -c.k[0]
    c.fill_all()
    c.upload()
    Call(c, F32, 1, q=q, scale=0.5).launch().check()


def test_shared_pages(dev):
    """Two sequences on the same pages, one of them shorter, and a table that names a page twice."""
    c = Case(dev, 39, F16, 4, 2, 64, 16, (64, 50, 48), (1, 1, 1)).fill_all()
    c.table[1] = c.table[0]
    c.table[2, 2] = c.table[2, 0]
    c.upload()
    Call(c, F32, 1).launch().check()


def test_offsets_over_4_gib(dev):
    n_pages = 20_000
    size = dev.kv_bytes(F16, 8, 128, 128, n_pages)
    pb = size // n_pages
    c = Case(dev, 41, F16, 16, 8, 128, 128, (300, 70), (1, 1), spare=0, shuffle=False).fill_all()
    far = {0: 19_999, 1: 16_385, 2: 17_000, 3: 18_001}
    K, V = dev.DevBuf(size), dev.DevBuf(size)
    for near, to in far.items():
        assert to * pb > 1 << 32
        K.upload(c.K[near], to * pb)
        V.upload(c.V[near], to * pb)
    c.dtable, c.dlen = dev.DevBuf.of(np.array([[far[0], far[1], far[2]], [far[3], -1, -1]], np.int32)), dev.DevBuf.of(np.array(c.lens, np.int32))
    c.kv = dev.Kv(F16, 8, 128, 128, n_pages, K, V, 2, 3, c.dtable, c.dlen)
    Call(c, F32, 1).launch().check()
    K.free(), V.free()


def test_graph_streams_and_workspaces(dev):
    """A captured call replayed while the lengths move on, beside another graph of other sizes on another stream with a workspace of its
    own; then both on one stream with one workspace."""
    a = Case(dev, 43, F16, 8, 2, 128, 16, (900, 40), (1, 1)).fill_all().upload()
    b = Case(dev, 44, F16, 16, 1, 64, 32, (3000, 700, 5), (2, 2, 2)).fill_all().upload()
    ca, cb = Call(a, F32, 1), Call(b, F16, 2)
    sa, sb = dev.Stream(), dev.Stream()
    ga, gb = dev.Graph(sa, lambda st: ca.launch(st)), dev.Graph(sb, lambda st: cb.launch(st))
    eager = cb.launch().check()
    for step in range(3):
        lens = [800 + 50 * step, 10 + 15 * step]
        a.dlen.upload(np.array(lens, np.int32))
        cb.Y.fill(0x5A)
        for _ in range(4):
            ga.launch(), gb.launch()
        sa.sync(), sb.sync()
        assert np.array_equal(cb.check(), eager)
        a.lens = lens
        ca.check()
    ws = dev.DevBuf(max(ca.size, cb.size))
    ws.fill(0)
    for _ in range(5):
        ca.launch(sa.s, ws), cb.launch(sa.s, ws)
    sa.sync()
    ca.check()
    assert np.array_equal(cb.check(), eager)
    assert not ws.download(np.uint32, 16384).any()


def test_same_bits_every_time(dev):
    c = Case(dev, 45, F16, 24, 4, 256, 64, (30_000,), (1,)).fill_all().upload()
    a = Call(c, F32, 1)
    first = a.launch().got()
    for _ in range(20):
        assert np.array_equal(a.launch().got(), first)


def test_what_the_device_refuses(dev):
    """A page outside the pool and a length that cannot be: NaN in that sequence's rows, the others right, and kv_check says so."""
    for message, page, n in (("page outside", 999, None), ("page outside", -1, None), ("length", None, 5000), ("length", None, -3), ("length", None, 1)):
        c = Case(dev, 47, F16, 4, 2, 64, 16, (2000, 60, 1200), (2, 2, 2)).fill_all()
        if page is not None:
            c.table[0, 70] = page
        c.upload()
        if n is not None:
            c.dlen.upload(np.array([n, 60, 1200], np.int32))
        a = Call(c, F32, 2)
        y = a.launch().got()
        with pytest.raises(dev.AmdcError, match=message):
            dev.kv_check()
        dev.kv_check()
        assert np.isnan(y[:2]).all() and np.isfinite(y[2:]).all()
        for b in (1, 2):
            k, v = c.stored(b)
            L = c.lens[b]
            want, av, aq = attn64(a.q[2 * b:2 * b + 2], k, v, float(a.scale), [L - 2, L - 1], 0)
            assert (np.abs(y[2 * b:2 * b + 2] - want) <= bound(c, F32, want, av, aq, L)).all()
        assert not a.ws.download(np.uint32, 16384).any()


def test_recording_refuses(dev):
    """The chain recorder has no such operation: the call is refused on the recording stream, nothing runs."""
    c = Case(dev, 49, F16, 4, 2, 64, 16, (20,), (1,)).fill_all().upload()
    a = Call(c, F32, 1)
    s = dev.Stream()
    with pytest.raises(dev.AmdcError, match="cannot be recorded"):
        with dev.ChainRecorder(s):
            a.launch(s.s)
    dev.sync()
    assert np.all(a.Y.download(np.uint8) == 0x5A)
