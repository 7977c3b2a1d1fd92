"""amdc_kv_append: keys (rotated) and values into the paged cache, and the rotated queries, against the definition in 64 bits;
everything else in the pools and behind the rows is left bit for bit. Positions, pages, rows and refusals."""
import numpy as np
import pytest

from attncase import BF16, F16, F32, TINY, ULP, Case, as_float, from16, rope64

pytestmark = pytest.mark.gpu


def freqs(n_rot, base=10000.0):
    return (base ** (-np.arange(0, n_rot, 2) / n_rot)).astype(np.float32)


def run(c, qt, mode, n_rot, pad=0, off=0, in_place=False, stream=None, with_q=True, freq=None):
    """Appends c's new rows: a fused row [q | k | v | pad values], starting `off` floats into the buffer. Returns what the cache
    and qo held before and hold after, and the inputs."""
    dev, g = c.dev, c.g
    wq, wk = c.n_q * c.hd, c.n_kv * c.hd
    w = wq + 2 * wk + pad
    x = g.standard_normal(off + c.total * w).astype(np.float32)
    X = dev.DevBuf.of(x)
    x = x[off:].reshape(c.total, w)
    f = freqs(n_rot) if freq is None else freq
    Fr = dev.DevBuf.of(f)
    qos = w if in_place else wq + (pad if qt == F32 else 2 * pad)
    esz = 4 if qt == F32 else 2
    QO = X if in_place else dev.DevBuf((off + c.total * qos) * esz)
    if not in_place:
        QO.fill(0x5A)
    before = QO.download(np.uint8).copy()
    qo = QO.ptr + off * esz
    dev.kv_append(c.kv, X.ptr + 4 * (off + wq), X.ptr + 4 * (off + wq + wk), X.ptr + 4 * off if with_q else None, qo if with_q else None, qt, c.n_q, c.T, w, w, w, qos,
                  cu=c.dcu if c.ragged else None, freq=Fr, n_rot=n_rot, rope=mode, stream=stream)
    return x, f, QO, before, qos, off


def check(c, qt, mode, n_rot, got, with_q=True):
    x, f, QO, before, qos, off = got
    dev = c.dev
    wq, wk = c.n_q * c.hd, c.n_kv * c.hd
    if c.dev is not None:
        dev.sync()
    K, V = c.dK.download(np.uint16).reshape(c.K.shape), c.dV.download(np.uint16).reshape(c.V.shape)
    wantK, wantV = c.K.copy(), c.V.copy()
    raw = QO.download(np.float32 if qt == F32 else np.uint16)[off:]
    raw0 = before.view(np.float32 if qt == F32 else np.uint16)[off:]
    kept = np.ones(len(raw), bool)
    for b in range(c.n_seq):
        L, m, r0 = c.lens[b], c.new[b], int(c.cu[b])
        if L == 0:
            continue
        rows = np.arange(r0, r0 + m)
        pos = np.arange(L - m, L)
        k, ke = rope64(x[rows, wq:wq + wk].reshape(m, c.n_kv, c.hd), pos, f, n_rot, mode)
        q, qe = rope64(x[rows, :wq].reshape(m, c.n_q, c.hd), pos, f, n_rot, mode)
        v = x[rows, wq + wk:wq + 2 * wk].reshape(m, c.n_kv, c.hd).astype(np.float64)
        for i, p in enumerate(pos):
            pg, s = c.table[b, p // c.page], p % c.page
            for name, pool, want, val, err in (("k", K, wantK, k[i], ke[i]), ("v", V, wantV, v[i], 0.0)):
                ix = (pg, slice(None), s // 16, slice(None), s % 16) if name == "k" else (pg, slice(None), s // 8, slice(None), s % 8)
                have = pool[ix].reshape(c.n_kv, c.hd)
                tol = ULP[c.type] * (np.abs(val) + err) + err + TINY[c.type]
                bad = ~(np.abs(from16(have, c.type) - val) <= tol)
                assert not bad.any(), f"{name} of sequence {b}, position {p}: {int(bad.sum())} values off"
                want[ix] = pool[ix]
        if with_q:
            for i, r in enumerate(rows):
                have = as_float(raw[r * qos:r * qos + wq], qt).reshape(c.n_q, c.hd)
                tol = ULP[qt] * (np.abs(q[i]) + qe[i]) + qe[i] + TINY[qt]
                bad = ~(np.abs(have - q[i]) <= tol)
                assert not bad.any(), f"query row {r}: {int(bad.sum())} values off"
                kept[r * qos:r * qos + wq] = False
    assert np.array_equal(K, wantK) and np.array_equal(V, wantV), "something else in the pools changed"
    assert np.array_equal(raw.view(np.uint32 if qt == F32 else np.uint16)[kept], raw0.view(np.uint32 if qt == F32 else np.uint16)[kept]), "something else in qo changed"
    dev.kv_check()


CASES = [
    # type, qt, n_q, n_kv, hd, page, mode, n_rot, lens, new, room, pad, off
    (F16, F32, 8, 8, 128, 64, 1, 128, (1,), (1,), 0, 0, 0),  # the first token of all
    (F16, F32, 32, 32, 128, 64, 1, 128, (700,), (1,), 0, 0, 0),
    (BF16, BF16, 24, 4, 256, 32, 2, 64, (65, 64, 63, 2, 1, 0, 333), (1,) * 7, 0, 0, 0),  # one of no part
    (F16, F16, 8, 2, 128, 16, 2, 128, (100, 37, 16), (100, 20, 16), 0, 0, 0),  # whole prompts and a chunk
    (BF16, F32, 6, 2, 64, 16, 1, 32, (29, 50, 8, 17), (9, 0, 8, 1), 5, 0, 0),  # an empty one; room behind the last
    (F16, F32, 4, 4, 64, 128, 2, 20, (131, 140), (7, 7), 0, 3, 1),  # a half that is no multiple of 8, unaligned rows
    (BF16, BF16, 2, 1, 256, 16, 1, 250, (40,), (23,), 0, 1, 1),
    (F16, F16, 7, 1, 128, 32, 0, 0, (33, 31), (2, 2), 0, 4, 0),  # no rotation
    (F16, F32, 40, 8, 128, 16, 2, 128, tuple(range(20, 20 + 70)), tuple(1 + i % 5 for i in range(70)), 0, 0, 0),  # over 64 sequences
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_append(dev, i):
    ty, qt, n_q, n_kv, hd, page, mode, n_rot, lens, new, room, pad, off = CASES[i]
    c = Case(dev, 100 + i, ty, n_q, n_kv, hd, page, lens, new, room=room).upload()
    check(c, qt, mode, n_rot, run(c, qt, mode, n_rot, pad, off))


def test_in_place(dev):
    """qo = q: the rotated queries over the queries, both kinds of pairs."""
    for mode in (1, 2):
        c = Case(dev, 7 + mode, F16, 24, 4, 256, 32, (70, 5, 300), (3, 3, 3)).upload()
        check(c, F32, mode, 64, run(c, F32, mode, 64, in_place=True))


def test_without_queries(dev):
    c = Case(dev, 9, BF16, 8, 8, 64, 16, (20, 9), (4, 4)).upload()
    check(c, F32, 2, 64, run(c, F32, 2, 64, with_q=False), with_q=False)


def test_far_positions(dev):
    """Angles of a million radians: f32 would keep a sixteenth of a turn of them."""
    c = Case(dev, 11, F16, 2, 1, 64, 65536, (1_500_007,), (3,), shuffle=False).upload()
    check(c, F32, 1, 64, run(c, F32, 1, 64))
    check(c, F32, 2, 32, run(c, F32, 2, 32))


def test_pool_over_4_gib(dev):
    """Pages whose offsets pass 32 bits."""
    n_pages = 20_000
    kv_bytes = dev.kv_bytes(F16, 8, 128, 128, n_pages)
    assert 16_385 * (kv_bytes // n_pages) > 1 << 32
    c = Case(dev, 12, F16, 8, 8, 128, 128, (200, 3), (130, 3), spare=0, shuffle=False)
    c.table[0, :2] = (19_999, 17_001)
    c.table[1, 0] = 16_385
    K, V = dev.DevBuf(kv_bytes), dev.DevBuf(kv_bytes)
    table, length, cu = dev.DevBuf.of(c.table), dev.DevBuf.of(np.array(c.lens, np.int32)), dev.DevBuf.of(c.cu)
    c.kv = dev.Kv(F16, 8, 128, 128, n_pages, K, V, 2, 2, table, length)
    c.dcu = cu
    x, f, *_ = run(c, F32, 2, 128)
    dev.kv_check()
    pb = kv_bytes // n_pages
    wq = wk = 8 * 128
    for b in range(2):
        for p in range(c.lens[b] - c.new[b], c.lens[b]):
            pg, s, r = int(c.table[b, p // 128]), p % 128, int(c.cu[b]) + p - (c.lens[b] - c.new[b])
            if p % 37 and p % 128 not in (0, 127):
                continue
            k = K.download(np.uint16, pb // 2, pg * pb).reshape(8, 8, 16, 16, 8)[:, s // 16, :, s % 16].reshape(8, 128)
            v = V.download(np.uint16, pb // 2, pg * pb).reshape(8, 16, 128, 8)[:, s // 8, :, s % 8]
            want, e = rope64(x[r:r + 1, wq:wq + wk].reshape(1, 8, 128), [p], f, 128, 2)
            assert (np.abs(from16(k, F16) - want[0]) <= ULP[F16] * (np.abs(want[0]) + e[0]) + e[0] + TINY[F16]).all()
            want = x[r, wq + wk:].reshape(8, 128).astype(np.float64)
            assert (np.abs(from16(v, F16) - want) <= ULP[F16] * np.abs(want) + TINY[F16]).all()
    K.free(), V.free()


def test_values_at_the_edges(dev):
    """Infinities, NaN and values over the type's range are stored as the conversion gives them, the neighbours unharmed."""
    c = Case(dev, 13, F16, 2, 2, 64, 16, (10,), (2,)).upload()
    x = np.ones((2, 6 * 64), np.float32)
    x[0, 4 * 64:4 * 64 + 5] = (np.inf, -np.inf, np.nan, 1e6, 1e-9)
    X = dev.DevBuf.of(x)
    dev.kv_append(c.kv, X.ptr + 4 * 128, X.ptr + 4 * 256, None, None, F32, 2, 2, 384, 384)
    V = c.dV.download(np.uint16).reshape(c.V.shape)[c.table[0, 0], 0, 1]
    got = from16(V[:5, 0], F16)
    assert got[0] == np.inf and got[1] == -np.inf and np.isnan(got[2]) and got[3] == np.inf and got[4] == 0
    assert (from16(V[5:, 0], F16) == 1).all() and (from16(V[:, 1], F16) == 1).all()


def test_what_the_device_refuses(dev):
    """A page outside the pool, a length over the table or under the new rows, rows outside T: nothing of that entry is written, the
    others are, and kv_check says so once."""
    def bad(message, lens=(20, 20), new=(2, 2), **change):
        c = Case(dev, 14, F16, 2, 2, 64, 16, (20, 20), new, ragged="cu" in change)
        if "page" in change:
            c.table[0, 1] = change["page"]
        if "cu" in change:
            c.cu[:] = change["cu"]
        c.upload()
        if lens != (20, 20):
            c.dlen.upload(np.array(lens, np.int32))
        x, f, *_ = run(c, F32, 1, 64)
        with pytest.raises(dev.AmdcError, match=message):
            dev.kv_check()
        dev.kv_check()
        K = c.dK.download(np.uint16).reshape(c.K.shape)
        changed = {int(p) for p in np.argwhere(K != c.K)[:, 0]}
        return changed, c
    for page in (4 + 2, -1, 0x7FFFFFFF, -(1 << 31)):
        changed, c = bad("page outside", page=page)
        assert changed == {int(c.table[1, 1])}
    for n in (33, 1, -5, 0x7FFFFFFF):
        changed, c = bad("length", lens=(n, 20))
        assert changed == {int(c.table[1, 1])}
    changed, c = bad("rows outside", new=(2, 1), cu=(0, 2, 9))
    assert changed == {int(c.table[0, 1])}
    bad("rows outside", new=(2, 1), cu=(-3, 2, 3))


def test_streams_and_graph(dev):
    """On a stream of its own, captured and replayed while the host moves the lengths on."""
    c = Case(dev, 15, F16, 4, 2, 128, 16, (14, 30), (1, 1)).upload()
    s = dev.Stream()
    w = (4 + 4) * 128
    x = c.g.standard_normal((2, w)).astype(np.float32)
    X, QO, Fr = dev.DevBuf.of(x), dev.DevBuf(2 * 4 * 128 * 4), dev.DevBuf.of(freqs(128))
    graph = dev.Graph(s, lambda st: dev.kv_append(c.kv, X.ptr + 4 * 512, X.ptr + 4 * 768, X, QO, F32, 4, 1, w, w, w, 512, freq=Fr, n_rot=128, rope=2, stream=st))
    for step in range(3):
        lens = np.array([14 + step, 30 + step], np.int32)
        c.dlen.upload(lens)
        graph.launch()
        s.sync()
        V = c.dV.download(np.uint16).reshape(c.V.shape)
        for b in range(2):
            p = int(lens[b]) - 1
            got = from16(V[c.table[b, p // 16], :, (p % 16) // 8, :, p % 8], F16)
            want = x[b, 768:].reshape(2, 128).astype(np.float64)
            assert (np.abs(got - want) <= ULP[F16] * np.abs(want) + TINY[F16]).all()
    dev.kv_check()
