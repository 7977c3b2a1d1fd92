"""The attention block of a layer as an engine runs it: RMSNorm + Q8, the fused qkv matrix, rotation and cache (queries in place), attention
with its Q8 copy, the output matrix with the residual. A prompt at once, a chunk of a second one, then decode and verify steps captured as
graphs and replayed while the host moves the lengths on. Every operator's result is checked on the inputs it had on the device."""
import numpy as np
import pytest

from amdc import synth
from attncase import F16, F32, TINY, ULP, Case, attn64, from16, rope64
from test_attn_decode import bound

pytestmark = pytest.mark.gpu
EPS = 1e-6


class Layer:
    """hidden 512, n_q heads over 2 of 64."""

    def __init__(self, dev, kind, rows):
        self.dev, self.kind, self.hd, self.n_q, self.n_kv, self.hidden, self.rows = dev, kind, 64, 8, 2, 512, rows
        self.w = (self.n_q + 2 * self.n_kv) * self.hd
        g = self.g = np.random.default_rng(71 + kind)
        self.W = dev.DevBuf.of(dev.repack(kind, synth.gguf(kind, self.w, self.hidden, 5), self.w, self.hidden))
        self.Wo = dev.DevBuf.of(dev.repack(kind, synth.gguf(kind, self.hidden, self.hidden, 6), self.hidden, self.hidden))
        self.norm = dev.DevBuf.of((1 + 0.1 * g.standard_normal(self.hidden)).astype(np.float32))
        self.freq_h = (10000.0 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32)
        self.freq = dev.DevBuf.of(self.freq_h)
        self.xs = (40 * 16 + 255) // 256 * 256
        self.X, self.N, self.Y = (dev.DevBuf(rows * self.hidden * 4) for _ in range(3))
        self.QKV, self.RAW = dev.DevBuf(rows * self.w * 4), dev.DevBuf(rows * self.w * 4)
        self.A, self.XQ, self.AQ = dev.DevBuf(rows * self.hidden * 4), dev.DevBuf(rows * self.xs), dev.DevBuf(rows * self.xs)
        for b in (self.XQ, self.AQ):
            b.fill(0)

    def run(self, kv, rows, T, ws, cu=None, decode=False, stream=None):
        """rows rows in all; T as the cache operators take it."""
        dev, h, w = self.dev, self.hidden, self.w
        dev.rmsnorm_q8(self.X, self.norm, self.N, h, EPS, self.XQ, rows, 4 * h, 4 * h, self.xs, stream=stream)
        dev.op_gemv(self.kind, self.W, self.XQ, self.QKV, w, 16, rows, self.xs, w, stream=stream)
        q = self.QKV.ptr
        dev.kv_append(kv, q + 4 * h, q + 4 * (h + 128), q, q, F32, self.n_q, T, w, w, w, w, cu=cu, freq=self.freq, n_rot=64, rope=dev.ROPE_HALVES, stream=stream)
        if decode:
            dev.attn_decode(kv, q, self.A, F32, self.n_q, T, w, h, 0.125, ws, ws.nbytes, q8=self.AQ, q8s=self.xs, stream=stream)
        else:
            dev.attn_prefill(kv, q, self.A, F32, self.n_q, T, w, h, 0.125, ws, ws.nbytes, cu=cu, q8=self.AQ, q8s=self.xs, stream=stream)
        dev.op_gemv(self.kind, self.Wo, self.AQ, self.Y, h, 16, rows, self.xs, h, h, res=self.X, stream=stream)

    def check(self, c, lens, new, orc):
        """The whole block after a run over c's sequences of lens positions, `new` rows each."""
        dev, h, w = self.dev, self.hidden, self.w
        rows = sum(new)
        dev.sync()
        dev.kv_check()
        dev.op_gemv(self.kind, self.W, self.XQ, self.RAW, w, 16, rows, self.xs, w)  # the qkv rows before the rotation
        raw = self.RAW.download(np.float32, rows * w).reshape(rows, w)
        qkv = self.QKV.download(np.float32, rows * w).reshape(rows, w)
        a = self.A.download(np.float32, rows * h).reshape(rows, h)
        c.K, c.V = c.dK.download(np.uint16).reshape(c.K.shape), c.dV.download(np.uint16).reshape(c.V.shape)
        r0 = 0
        for b, (L, m) in enumerate(zip(lens, new)):
            if m:
                c.lens[b] = L
                pos = np.arange(L - m, L)
                k, v = c.stored(b)
                x = raw[r0:r0 + m].astype(np.float64)
                want, e = rope64(x[:, h:h + 128].reshape(m, 2, 64), pos, self.freq_h, 64, 2)
                assert (np.abs(k[pos] - want) <= ULP[F16] * (np.abs(want) + e) + e + TINY[F16]).all()
                assert (np.abs(v[pos] - x[:, h + 128:].reshape(m, 2, 64)) <= ULP[F16] * np.abs(x[:, h + 128:].reshape(m, 2, 64)) + TINY[F16]).all()
                want, e = rope64(x[:, :h].reshape(m, 8, 64), pos, self.freq_h, 64, 2)
                q = qkv[r0:r0 + m, :h].reshape(m, 8, 64).astype(np.float64)
                assert (np.abs(q - want) <= e + 2.0 ** -24 * np.abs(want)).all()
                want, av, aq = attn64(q, k, v, 0.125, pos, 0)
                assert (np.abs(a[r0:r0 + m].reshape(m, 8, 64) - want) <= bound(c, F32, want, av, aq, L)).all(), f"sequence {b}"
            r0 += m
        aq = self.AQ.download(np.uint8).reshape(self.rows, self.xs)[:rows, :640]
        assert np.array_equal(aq, orc.quant_q8(a))
        y = self.Y.download(np.uint32, rows * h)
        dev.op_gemv(self.kind, self.Wo, self.AQ, self.Y, h, 16, rows, self.xs, h, h, res=self.X)
        assert np.array_equal(self.Y.download(np.uint32, rows * h), y)
        assert np.isfinite(y.view(np.float32)).all()


@pytest.mark.parametrize("kind", (synth.KIND_Q4_0, synth.KIND_Q4_K))
def test_layer(dev, orc, kind):
    layer = Layer(dev, kind, 64)
    c = Case(dev, 72, F16, 8, 2, 64, 16, (120, 90), (1, 1)).upload()  # room for what follows; the pools hold NaN
    ws = dev.DevBuf(max(dev.attn_prefill_ws(c.kv, 8, 64), dev.attn_decode_ws(c.kv, 8, 1), dev.attn_decode_ws(c.kv, 8, 3)))
    ws.fill(0)
    cu = dev.DevBuf(12)

    def feed(rows):
        layer.X.upload(layer.g.standard_normal((rows, 512)).astype(np.float32))

    # a prompt of 41 and the first 9 of another, packed
    feed(50)
    c.dlen.upload(np.array([41, 9], np.int32)), cu.upload(np.array([0, 41, 50], np.int32))
    layer.run(c.kv, 50, 50, ws, cu=cu)
    layer.check(c, [41, 9], [41, 9], orc)
    # the second one's next chunk alone
    feed(33)
    c.dlen.upload(np.array([41, 42], np.int32)), cu.upload(np.array([0, 0, 33], np.int32))
    layer.run(c.kv, 33, 33, ws, cu=cu)
    layer.check(c, [41, 42], [0, 33], orc)
    # decode steps, then verify steps of three tokens: captured, replayed on the lengths of the step
    s = dev.Stream()
    lens = [41, 42]
    for T, steps in ((1, 4), (3, 3)):
        layer.run(c.kv, 2 * T, T, ws, decode=True, stream=s.s)  # the GEMVs' workspaces of these sizes, before the capture
        s.sync()
        graph = dev.Graph(s, lambda st: layer.run(c.kv, 2 * T, T, ws, decode=True, stream=st))
        for _ in range(steps):
            feed(2 * T)
            lens = [n + T for n in lens]
            c.dlen.upload(np.array(lens, np.int32))
            graph.launch()
            s.sync()
            layer.check(c, lens, [T, T], orc)
        del graph
    assert not ws.download(np.uint32, 16384).any()
