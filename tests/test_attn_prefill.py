"""amdc_attn_prefill against the definition in 64 bits on the cache's stored values: prompts and chunks of different lengths packed, and
the uniform form. Positions that no row sees hold NaN (attncase.Case)."""
import numpy as np
import pytest

from attncase import BF16, F16, F32, ULP, Case, as_float, attn64, to16
from test_attn_decode import bound

pytestmark = pytest.mark.gpu


class Call:
    def __init__(self, c, t, window=0, scale=None, pad=0, off=0, q=None, q8=False, amp=2.0):
        dev, self.c, self.t, self.window = c.dev, c, t, window
        w = c.n_q * c.hd
        self.scale = np.float32(1 / np.sqrt(c.hd) if scale is None else scale)
        self.qs, self.ys, self.off, rows = w + pad, w + 2 * pad, off, c.total
        q = (amp * c.g.standard_normal((rows, w))).astype(np.float32) if q is None else q.reshape(rows, w).astype(np.float32)
        buf = np.full(off + rows * self.qs, np.nan, np.float32)
        buf[off:].reshape(rows, self.qs)[:c.rows, :w] = q[:c.rows]  # NaN in rows of no sequence
        raw = buf if t == F32 else to16(buf, t)
        self.q = as_float(raw, t)[off:].reshape(rows, self.qs)[:, :w].reshape(rows, c.n_q, c.hd)
        esz = self.esz = 4 if t == F32 else 2
        self.Q, self.Y = dev.DevBuf.of(raw), dev.DevBuf((off + rows * self.ys) * esz)
        self.Y.fill(0x5A)
        self.q8s = w // 32 * 40 + 4 * pad
        self.Q8 = dev.DevBuf(rows * self.q8s) if q8 else None
        if q8:
            self.Q8.fill(0xA5)
        self.size = dev.attn_prefill_ws(c.kv, c.n_q, rows)
        self.ws = dev.DevBuf(self.size)
        self.ws.fill(0)
        self.rows, self.w = rows, w

    def launch(self, stream=None, ws=None, y=True):
        c = self.c
        c.dev.attn_prefill(c.kv, self.Q.ptr + self.off * self.esz, self.Y.ptr + self.off * self.esz if y else None, self.t, c.n_q, c.T, self.qs, self.ys, self.scale,
                           (ws or self.ws), (ws or self.ws).nbytes, cu=c.dcu if c.ragged else None, window=self.window, q8=self.Q8, q8s=self.q8s if self.Q8 else 0,
                           stream=stream)
        return self

    def got(self):
        self.c.dev.sync()
        raw = self.Y.download(np.float32 if self.t == F32 else np.uint16)
        rows = raw[self.off:].reshape(self.rows, self.ys)
        untouched = np.concatenate([raw[:self.off].ravel(), rows[:, self.w:].ravel(), rows[self.c.rows:].ravel()])
        assert np.all(untouched.view(np.uint8) == 0x5A), "something beside the sequences' rows was written"
        return as_float(rows[:, :self.w].copy(), self.t).reshape(self.rows, self.c.n_q, self.c.hd)

    def check(self, lens=None, every=1):
        """every: of long sequences only every so many-th row is computed in 64 bits, and the last ones."""
        c = self.c
        y = self.got()
        lens = c.lens if lens is None else lens
        for b, L in enumerate(lens):
            m, r0 = c.new[b], int(c.cu[b])
            if not m:
                continue
            if L == 0:
                assert np.all(y[r0:r0 + m] == 0), f"sequence {b} of no positions"
                continue
            assert np.isfinite(y[r0:r0 + m]).all()
            k, v = c.stored(b)
            some = np.unique(np.concatenate([np.arange(0, m, every), np.arange(max(0, m - 3), m)]))
            want, av, aq = attn64(self.q[r0 + some], k, v, float(self.scale), L - m + some, self.window)
            off = np.abs(y[r0 + some] - want) / bound(c, self.t, want, av, aq, L)
            assert off.max() <= 1, f"sequence {b} of {L}, {m} new: {off.max():.2f} of the bound at {np.unravel_index(off.argmax(), off.shape)}, {int((~(off <= 1)).sum())} values"
        assert not self.ws.download(np.uint32, 16384).any(), "a counter was left"
        c.dev.kv_check()
        return y


CASES = [
    # type, t, n_q, n_kv, hd, page, window, lens, new, room
    (F16, F32, 4, 4, 128, 64, 0, (77,), (77,), 0),
    (F16, F16, 4, 4, 64, 16, 0, (1,), (1,), 0),
    (F16, F16, 2, 1, 64, 16, 0, (31, 32, 33, 63, 64, 65, 127, 128, 129), (31, 32, 33, 63, 64, 65, 127, 128, 129), 0),
    (BF16, BF16, 8, 2, 128, 32, 0, (300, 5, 170, 64), (300, 5, 30, 0), 7),  # a prompt, a chunk, a sequence without new rows; room behind
    (F16, F32, 6, 1, 256, 64, 0, (1500,), (40,), 0),  # a short chunk at the end: split
    (BF16, F32, 5, 1, 128, 16, 0, (200, 0, 90), (50, 20, 90), 0),  # one of no part
    (F16, F16, 4, 2, 128, 128, 0, (700,), (700,), 0),
    (BF16, F32, 3, 3, 64, 32, 50, (260, 51, 300), (260, 51, 100), 3),  # a window
    (F16, F32, 12, 2, 64, 16, 1, (130, 64), (130, 10), 0),  # of the row itself
    (BF16, BF16, 2, 2, 256, 16, 130, (500, 129), (500, 129), 0),
    (BF16, F32, 4, 1, 256, 16, 0, (150, 290), (150, 20), 0),
    (F16, F16, 7, 1, 256, 32, 0, (97,), (97,), 0),
    (F16, F32, 128, 1, 64, 16, 0, (9, 40), (9, 2), 0),  # 128 heads on one: a token is a tile
    (F16, F16, 100, 1, 64, 16, 40, (60,), (33,), 0),
    (F16, F32, 2, 2, 128, 16, 0, tuple(3 + 7 * i % 60 for i in range(80)), tuple(1 + i % 3 for i in range(80)), 0),  # over 64 sequences
    (F16, F32, 8, 2, 64, 16, 0, (40, 9, 128), (8, 8, 8), 0),  # uniform: cu NULL
    (BF16, BF16, 4, 4, 128, 16, 0, (200, 150), (150, 150), 0),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_prefill(dev, i):
    ty, t, n_q, n_kv, hd, page, window, lens, new, room = CASES[i]
    print(CASES[i], flush=True)
    c = Case(dev, 400 + i, ty, n_q, n_kv, hd, page, lens, new, room=room).fill_all().upload()
    Call(c, t, window).launch().check()


@pytest.mark.parametrize("ty,t,hd", [(F16, F16, 64), (F16, F32, 128), (BF16, BF16, 128), (F16, F32, 256), (BF16, F32, 256)])
def test_long(dev, ty, t, hd):
    """Thousands of positions; the tables of a wave's tiles are read again every 64."""
    c = Case(dev, 430 + hd, ty, 2, 1, hd, 16, (9000, 4500), (333, 200)).fill_all().upload()
    Call(c, t).launch().check(every=41)
    Call(c, t, window=4300).launch().check(every=41)


def test_equal_to_decode(dev):
    """A chunk of five rows by either operator: the same within the bound of both."""
    c = Case(dev, 440, F16, 24, 4, 256, 64, (900, 333), (5, 5)).fill_all().upload()
    Call(c, F32).launch().check()


@pytest.mark.parametrize("t", (F32, BF16))
def test_rows_that_are_not_aligned(dev, t):
    c = Case(dev, 441, BF16, 4, 2, 128, 16, (70, 300), (70, 40)).fill_all().upload()
    Call(c, t, pad=3, off=1).launch().check()


@pytest.mark.parametrize("hd,lens,new", [(64, (70, 0, 33), (70, 4, 20)), (128, (200, 9), (200, 9)), (256, (40, 50), (40, 20)), (256, (3000, 9), (30, 9))])
def test_q8_copy(dev, orc, hd, lens, new):
    """The Q8 copy is amdc_quant_q8's of the f32 result, split or not, with y or without."""
    c = Case(dev, 450 + hd, F16, 4, 2, hd, 16, lens, new).fill_all().upload()
    a = Call(c, F32, q8=True, pad=1)
    y = a.launch().check().astype(np.float32).reshape(a.rows, a.w)
    want = orc.quant_q8(y)
    for again in range(2):
        got = a.Q8.download(np.uint8).reshape(a.rows, a.q8s)
        assert np.array_equal(got[:, :want.shape[1]], want)
        assert np.all(got[:, want.shape[1]:] == 0xA5)
        a.Q8.fill(0xA5)
        a.launch(y=False)
        dev.sync()


def test_infinities_where_rows_do_not_see(dev):
    """A prompt in which one position's value is infinite and a later one's NaN: the rows before each are as if it were not there."""
    for ty, t, hd in ((F16, F16, 128), (F16, F32, 64), (BF16, F32, 128), (BF16, BF16, 256), (F16, F32, 256)):
        c = Case(dev, 460 + hd, ty, 4, 2, hd, 16, (150, 70), (150, 30)).fill_all()
        for b, (L, p1, p2) in enumerate(((150, 70, 101), (70, 45, 69))):
            v = c.v[b].copy()
            v[p1, :, 5], v[p2, :, 7] = np.inf, np.nan
            c.put(b, 0, L, None, v)
        c.upload()
        a = Call(c, t).launch()
        y = a.got()
        for b, (L, p1, p2) in enumerate(((150, 70, 101), (70, 45, 69))):
            m, r0 = c.new[b], int(c.cu[b])
            k, v = c.stored(b)
            pos = np.arange(L - m, L)
            want, av, aq = attn64(a.q[r0:r0 + m], k, np.where(np.isfinite(v), v, 0.0), float(a.scale), pos, 0)
            off = np.abs(y[r0:r0 + m] - want) / bound(c, t, want, av, aq, L)
            off[pos >= p1, :, 5] = 0
            off[pos >= p2, :, 7] = 0
            assert off.max() <= 1, (ty, t, hd, b)
            assert not np.isfinite(y[r0:r0 + m][pos >= p1, :, 5]).any() and np.isnan(y[r0:r0 + m][pos >= p2, :, 7]).all()


def test_keys_where_rows_do_not_see(dev):
    """A NaN key: the rows before its position are as if it were not there, its own and later ones NaN; with a window, those past it right
    again."""
    c = Case(dev, 470, F16, 2, 1, 64, 16, (200,), (200,)).fill_all()
    k = c.k[0].copy()
    k[90, :, 3] = np.nan
    c.put(0, 90, 91, k, None)
    c.upload()
    for t in (F32, F16):
        a = Call(c, t, window=60).launch()
        y = a.got()
        ks, vs = c.stored(0)
        pos = np.arange(200)
        ok = (pos < 90) | (pos >= 150)
        want, av, aq = attn64(a.q[ok], np.nan_to_num(ks), vs, float(a.scale), pos[ok], 60)
        assert (np.abs(y[ok] - want) <= bound(c, t, want, av, aq, 200)).all()
        assert np.isnan(y[~ok]).all()


@pytest.mark.parametrize("ty,hd,page,lens,new", [(F16, 64, 16, (300, 77, 700), (20, 9, 70)), (BF16, 128, 32, (300, 77, 3000), (20, 9, 3)), (F16, 256, 16, (300, 77, 5000), (20, 1, 4))])
def test_pages_before_the_window(dev, ty, hd, page, lens, new):
    """Entries of pages that are wholly before every row's window, given back to the pool, may be anything."""
    window = 40
    c = Case(dev, 471, ty, 4, 2, hd, page, lens, new).fill_all().upload()
    gone = c.table.copy()
    for b, L in enumerate(lens):
        gone[b, :max(0, L - new[b] + 1 - window) // page] = (-1, 999999, -2 ** 31)[b]
    c.dtable.upload(gone)
    for t in (F32, ty):
        Call(c, t, window=window).launch().check()
    dev.kv_check()


def test_extreme_scores(dev):
    c = Case(dev, 480, F16, 4, 2, 128, 16, (100, 33), (100, 20)).fill_all().upload()
    q = c.g.standard_normal((120, 4 * 128))
    Call(c, F32, q=q * 1e9, scale=1e-9 / 11).launch().check()
    Call(c, F32, q=q * 1e-30, scale=1e30 / 11).launch().check()
    Call(c, F32, q=q * 0).launch().check()
    Call(c, F32, q=q * 40).launch().check()
    Call(c, F16, q=q * 40).launch().check()
    Call(c, F32, q=q, scale=-0.3).launch().check()
    c = Case(dev, 481, F16, 2, 2, 64, 16, (500,), (500,))
    c.k[0][:] = (np.arange(500) / 80 - 3)[:, None, None] + 0.01 * c.k[0]  # the maximum is raised again and again
    c.fill_all().upload()
    Call(c, F32, q=np.ones((500, 128)), scale=0.5).launch().check(every=7)
    Call(c, F16, q=np.ones((500, 128)), scale=0.5).launch().check(every=7)


def test_scales_of_zero_and_near_it(dev):
    """Scale 0 is the mean, whatever the products; a subnormal scale of products near f32's largest."""
    c = Case(dev, 482, BF16, 4, 2, 64, 16, (100, 33), (100, 20), amp=1e18).fill_all().upload()
    q = c.g.standard_normal((120, 4 * 64))
    for t in (F32, BF16):
        Call(c, t, q=q * 1e18, scale=0.0).launch().check()
        Call(c, t, q=q * 1e18, scale=1e-39).launch().check()
    c = Case(dev, 483, F16, 4, 2, 128, 16, (100, 33), (100, 20)).fill_all().upload()
    Call(c, F32, scale=0.0, window=30).launch().check()
    Call(c, F16, scale=0.0).launch().check()


def test_offsets_over_4_gib(dev):
    n_pages = 20_000
    size = dev.kv_bytes(BF16, 8, 128, 128, n_pages)
    pb = size // n_pages
    c = Case(dev, 482, BF16, 8, 8, 128, 128, (300, 70), (60, 70), spare=0, shuffle=False).fill_all()
    far = {0: 19_999, 1: 16_385, 2: 17_000, 3: 18_001}
    K, V = dev.DevBuf(size), dev.DevBuf(size)
    for near, to in far.items():
        assert to * pb > 1 << 32
        K.upload(c.K[near], to * pb)
        V.upload(c.V[near], to * pb)
    c.dtable, c.dlen, c.dcu = dev.DevBuf.of(np.array([[far[0], far[1], far[2]], [far[3], -1, -1]], np.int32)), dev.DevBuf.of(np.array(c.lens, np.int32)), dev.DevBuf.of(c.cu)
    c.kv = dev.Kv(BF16, 8, 128, 128, n_pages, K, V, 2, 3, c.dtable, c.dlen)
    Call(c, BF16).launch().check(every=3)
    K.free(), V.free()


def test_graph_streams_and_workspaces(dev):
    """A captured call replayed while lengths and rows move, beside another on another stream with a workspace of its own; then both, and
    a decode, on one stream with one workspace."""
    a = Case(dev, 484, F16, 8, 2, 128, 16, (900, 40), (20, 12), room=8).fill_all().upload()
    b = Case(dev, 485, F16, 16, 1, 64, 32, (3000, 700, 5), (2, 2, 2)).fill_all().upload()
    ca, cb = Call(a, F32), Call(b, F16)
    sa, sb = dev.Stream(), dev.Stream()
    ga, gb = dev.Graph(sa, lambda st: ca.launch(st)), dev.Graph(sb, lambda st: cb.launch(st))
    eager = cb.launch().check()
    for step in range(3):
        lens, new = [800 + 50 * step, 10 + 15 * step], [20 - 3 * step, 3 + step]
        a.dlen.upload(np.array(lens, np.int32))
        a.new, a.rows = new, sum(new)
        a.cu = np.array([0, new[0], sum(new)], np.int32)
        a.dcu.upload(a.cu)
        q = np.random.default_rng(step)
        x = q.standard_normal((ca.rows, ca.w)).astype(np.float32)
        ca.Q.upload(x)
        ca.q = x.astype(np.float64).reshape(ca.q.shape)
        ca.Y.fill(0x5A)
        cb.Y.fill(0x5A)
        for _ in range(4):
            ga.launch(), gb.launch()
        sa.sync(), sb.sync()
        assert np.array_equal(cb.check(), eager)
        ca.check(lens)
    ws = dev.DevBuf(max(ca.size, cb.size, dev.attn_decode_ws(b.kv, 16, 2)))
    ws.fill(0)
    Y = dev.DevBuf(6 * 16 * 64 * 2)
    for _ in range(5):
        ca.launch(sa.s, ws), cb.launch(sa.s, ws)
        dev.attn_decode(b.kv, cb.Q, Y, F16, 16, 2, 1024, 1024, cb.scale, ws, ws.nbytes, stream=sa.s)
    sa.sync()
    ca.check(lens)
    assert np.array_equal(cb.check(), eager)
    assert not ws.download(np.uint32, 16384).any()
    d = as_float(Y.download(np.uint16), F16).reshape(6, 16, 64)
    for i, L in enumerate(b.lens):
        k, v = b.stored(i)
        want, av, aq = attn64(cb.q[2 * i:2 * i + 2], k, v, float(cb.scale), [L - 2, L - 1], 0)
        assert (np.abs(d[2 * i:2 * i + 2] - want) <= bound(b, F16, want, av, aq, L)).all()


def test_same_bits_every_time(dev):
    c = Case(dev, 486, F16, 6, 1, 256, 64, (6000,), (21,)).fill_all().upload()
    a = Call(c, F32)
    first = a.launch().got()
    for _ in range(20):
        assert np.array_equal(a.launch().got(), first)


def test_what_the_device_refuses(dev):
    for message, page, n in (("page outside", 999, None), ("page outside", -1, None), ("length", None, 5000), ("length", None, -3), ("length", None, 10)):
        c = Case(dev, 488, F16, 4, 2, 64, 16, (2000, 60, 1200), (20, 60, 30)).fill_all()
        if page is not None:
            c.table[0, 70] = page
        c.upload()
        if n is not None:
            c.dlen.upload(np.array([n, 60, 1200], np.int32))
        a = Call(c, F32)
        y = a.launch().got()
        with pytest.raises(dev.AmdcError, match=message):
            dev.kv_check()
        dev.kv_check()
        assert np.isnan(y[:20]).all() and np.isfinite(y[20:]).all()
        for b in (1, 2):
            k, v = c.stored(b)
            L, m, r0 = c.lens[b], c.new[b], int(c.cu[b])
            want, av, aq = attn64(a.q[r0:r0 + m], k, v, float(a.scale), np.arange(L - m, L), 0)
            assert (np.abs(y[r0:r0 + m] - want) <= bound(c, F32, want, av, aq, L)).all()
        assert not a.ws.download(np.uint32, 16384).any()
    # rows outside T: that sequence is left out, the ones that can be are computed
    c = Case(dev, 489, F16, 4, 2, 64, 16, (60, 70), (10, 5)).fill_all().upload()
    a = Call(c, F32)
    c.dcu.upload(np.array([0, 10, 400], np.int32))
    a.launch()
    dev.sync()
    with pytest.raises(dev.AmdcError, match="rows outside"):
        dev.kv_check()
    y = a.Y.download(np.uint32).reshape(15, -1)
    assert (y[10:] == 0x5A5A5A5A).all()
    k, v = c.stored(0)
    want, av, aq = attn64(a.q[:10], k, v, float(a.scale), np.arange(50, 60), 0)
    assert (np.abs(y[:10].view(np.float32).astype(np.float64).reshape(10, 4, 64) - want) <= bound(c, F32, want, av, aq, 60)).all()
