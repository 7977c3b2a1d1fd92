"""The linear-attention block of a layer as an engine runs it: the matrix of q, k, v, z and the gates, the convolution, the delta rule, the
gated norm with its Q8 copy, the output matrix, and the norms around the residual, whose Q8 copy the next matrix takes. Two prompts packed, a
chunk of the second alone, then decode steps (states in place) and verify steps (a state after every token, the next step from the one of the
token that was accepted), captured as graphs and replayed while the host moves the slots. Every operator's result is checked on the
inputs it had on the device."""
import numpy as np
import pytest

import lincase
from amdc import synth
from attncase import F32, TINY
from lincase import U, conv64, near, pool_of, sigmoid, state_of

pytestmark = pytest.mark.gpu
EPS = 1e-6
N_K, N_V, DK, DV, HIDDEN, SLOTS = 2, 4, 64, 64, 512, 13
CH, VAL = 2 * N_K * DK + N_V * DV, N_V * DV
W = CH + VAL + 16  # q k v | z | a b and 8 that nobody reads
SCALE = 0.5  # of the block in the residual
FLUSH = 2.0 ** -126  # a sigmoid under the smallest normal is 0: what it is multiplied by, times this, is lost


class Layer:
    def __init__(self, dev, kind, rows):
        self.dev, self.kind, self.rows = dev, kind, rows
        g = self.g = np.random.default_rng(81 + kind)
        f32 = lambda *s: g.standard_normal(s).astype(np.float32)
        up = lambda x: dev.DevBuf.of(np.ascontiguousarray(x, np.float32))
        self.Wi = dev.DevBuf.of(dev.repack(kind, synth.gguf(kind, W, HIDDEN, 5), W, HIDDEN))
        self.Wo = dev.DevBuf.of(dev.repack(kind, synth.gguf(kind, HIDDEN, VAL, 6), HIDDEN, VAL))
        self.wc, self.bias = f32(CH, 4) / 2, f32(CH)
        self.wn, self.w1, self.w2 = 1 + f32(DV) / 8, 1 + f32(HIDDEN) / 8, 1 + f32(HIDDEN) / 8
        self.dwc, self.dbias, self.dwn, self.dw1, self.dw2 = up(self.wc), up(self.bias), up(self.wn), up(self.w1), up(self.w2)
        self.L = lincase.Layer(g, rows, N_K, N_V, DK, DV, tiled=True, eps=EPS)
        self.dA, self.ddt = up(self.L.A), up(self.L.dt)
        self.gdn = dev.Gdn(N_K, N_V, DK, DV, dev.HEADS_TILED, float(self.L.scale), EPS, self.dA, self.ddt)
        self.qx, self.qv = (HIDDEN // 32 * 40 + 255) // 256 * 256, (VAL // 32 * 40 + 255) // 256 * 256
        buf = lambda n: dev.DevBuf(rows * 4 * n)
        self.X, self.P, self.Cv, self.G, self.A, self.Y, self.N = buf(HIDDEN), buf(W), buf(CH), buf(VAL), buf(VAL), buf(HIDDEN), buf(HIDDEN)
        self.XQ, self.AQ = dev.DevBuf(rows * self.qx), dev.DevBuf(rows * self.qv)
        self.XQ.fill(0), self.AQ.fill(0)
        self.pc, self.ps = dev.DevBuf(dev.conv_bytes(CH, 4, SLOTS)), dev.DevBuf(dev.gdn_bytes(N_V, DK, DV, SLOTS))
        self.pc.fill(0xFF), self.ps.fill(0xFF)  # NaN: no slot is read before it is written
        self.start, self.to, self.cu = (dev.DevBuf.of(np.full(8, -1, np.int32)) for _ in range(3))
        self.slots = dev.Slots(2, SLOTS, self.start, self.to)
        self.ws = dev.DevBuf(dev.gdn_prefill_ws(self.gdn, 2, rows))

    def feed(self, rows, start, to, cu=None):
        """What a step starts from: the residual rows, the Q8 copy that the norm before left, the slots."""
        self.x = self.g.standard_normal((rows, HIDDEN)).astype(np.float32)
        self.X.upload(self.x)
        self.dev.rmsnorm_q8(self.X, self.dw2, self.N, HIDDEN, EPS, self.XQ, rows, 4 * HIDDEN, 4 * HIDDEN, self.qx)
        self.start.upload(np.array(start, np.int32)), self.to.upload(np.array(to, np.int32))
        if cu is not None:
            self.cu.upload(np.array(cu, np.int32))
        self.dev.sync()
        self.hc, self.hs = self.pools()
        self.at = start, to

    def pools(self):
        return self.pc.download(np.float32).reshape(SLOTS, 3, CH), state_of(self.ps.download(np.float32).reshape(SLOTS, N_V, DV // 16, DK, 16))

    def run(self, rows, T, cu=None, decode=False, each=0, stream=None):
        d, p = self.dev, self.P.ptr
        d.op_gemv(self.kind, self.Wi, self.XQ, self.P, W, HIDDEN // 32, rows, self.qx, W, stream=stream)
        d.conv(self.slots, self.pc, self.P, self.dwc, self.dbias, self.Cv, F32, CH, 4, T, W, CH, cu=cu, each=each, stream=stream)
        q, ab = self.Cv.ptr, p + 4 * (CH + VAL)
        args = (self.gdn, self.slots, self.ps, q, q + 4 * N_K * DK, q + 8 * N_K * DK, ab, ab + 4 * N_V, self.G, F32, T, CH, CH, CH, W, W, VAL)
        if decode:
            d.gdn_decode(*args, each=each, stream=stream)
        else:
            d.gdn_prefill(*args, self.ws, self.ws.nbytes, cu=cu, stream=stream)
        d.norm_gate_q8(self.G, F32, self.dwn, p + 4 * CH, self.A, N_V, DV, EPS, d.GATE_SILU, self.AQ, rows, 4 * VAL, 4 * W, 4 * VAL, self.qv, stream=stream)
        d.op_gemv(self.kind, self.Wo, self.AQ, self.Y, HIDDEN, VAL // 32, rows, self.qv, HIDDEN, stream=stream)
        d.norm_res_q8(self.Y, self.dw1, SCALE, self.X, self.X, self.dw2, self.N, HIDDEN, EPS, self.XQ, rows, 4 * HIDDEN, 4 * HIDDEN, 4 * HIDDEN, 4 * HIDDEN, self.qx, stream=stream)

    def floor(self, rows, S):
        """What run64's bound, which grows and shrinks with the tokens, lacks where some of a sequence's values are much smaller than others
        (SiLU's of very negative numbers, states that a gate has all but cleared). A column of a chunk is scaled by one power of two, which
        brings m = 12 max |S| + 65 max |v|, S and v of this chunk and the one before, into [2^6, 2^7); its values times 2^8 are two f16
        parts, whose last place is 2^-24: off by up to 2^-25 2^-8 2^-6 m = 2^-39 m. A u is a sum of 64 of them, a y and an entry of the new state
        ones of 64 u, with factors up to 1 (|q^| = scale) and errors of either sign: 2^-39 8 8 m = 2^-33 m, and m is at most 77 of the
        larger of max |S| and max |v|: under 2^-26 of that."""
        v = np.abs(rows[:, 2 * N_K * DK:].reshape(-1, N_V, DV).astype(np.float64)).max(0)
        return 2.0 ** -26 * np.maximum(v, np.abs(np.array(S)).max((0, 2)))

    def check(self, new, orc, decode=False, each=False):
        d, rows = self.dev, sum(new)
        d.sync()
        d.kv_check()
        get = lambda b, n: b.download(np.float32, rows * n).reshape(rows, n)
        P, Cv, G, A, Y, X, N = get(self.P, W), get(self.Cv, CH), get(self.G, VAL), get(self.A, VAL), get(self.Y, HIDDEN), get(self.X, HIDDEN), get(self.N, HIDDEN)
        pc, ps = self.pools()
        start, to = self.at
        wc, ws, es = self.hc.astype(np.float64), self.hs.astype(np.float64), np.zeros(self.hs.shape)
        self.L.x, self.L.ab = Cv.astype(np.float64), np.ascontiguousarray(P[:, CH + VAL:CH + VAL + 2 * N_V + 1])
        r0, k = 0, 0
        for b, m in enumerate(new):
            if not m:
                continue
            sl = slice(r0, r0 + m)
            old = self.hc[start[b]] if start[b] >= 0 else np.zeros((3, CH))
            want, mag, pre, st = conv64(P[sl, :CH], self.wc, self.bias, old, 1)
            near(Cv[sl], want, U * 5 * mag * 1.2 + U * (6 + 2 * np.abs(pre)) * np.abs(want) + FLUSH * np.abs(pre) + TINY[F32], f"convolution {b}")  # as in test_conv
            old = self.hs[start[b]] if start[b] >= 0 else np.zeros((N_V, DK, DV), np.float32)
            want, err, S, E = self.L.run64(sl, old, chunk=1 if decode else 64)
            # subnormal values: half a step for each of 64 products of k S and of q S, and of less than as many operations on u and S
            floor = np.full((N_V, DV), 256 * TINY[F32]) + (0 if decode else self.floor(Cv[sl], [old] + S))
            near(G[sl].reshape(m, N_V, DV), want, err + U * np.abs(want) + floor, f"delta rule {b}")
            for t in range(m) if each else [m - 1]:
                o = to[r0 + t if each else b]
                wc[o], ws[o], es[o] = st[t], S[t], E[t] + floor[:, None]
            r0 += m
        assert np.array_equal(pc, wc.astype(np.float32), equal_nan=True)
        near(ps.astype(np.float64), ws, es, "states")
        g, z = G.astype(np.float64).reshape(rows, N_V, DV), P[:, CH:CH + VAL].astype(np.float64)
        want = (g / np.sqrt((g * g).mean(2, keepdims=True) + EPS) * self.wn).reshape(rows, VAL) * z
        # subnormal values: half a step for each of four products, times the factors behind it, |w| < 2 and |z|
        near(A.astype(np.float64), want * sigmoid(z), U * (20 + 2 * np.abs(z)) * np.abs(want * sigmoid(z)) + FLUSH * np.abs(want) + 8 * (1 + np.abs(z)) * TINY[F32], "gated norm")
        assert np.array_equal(self.AQ.download(np.uint8).reshape(self.rows, self.qv)[:rows, :VAL // 32 * 40], orc.quant_q8(A))
        again = d.DevBuf(rows * HIDDEN * 4)
        d.op_gemv(self.kind, self.Wo, self.AQ, again, HIDDEN, VAL // 32, rows, self.qv, HIDDEN)
        assert np.array_equal(again.download(np.float32).reshape(rows, HIDDEN), Y) and np.isfinite(Y).all()
        y = Y.astype(np.float64)
        y = SCALE * y / np.sqrt((y * y).mean(1, keepdims=True) + EPS) * self.w1
        near(X.astype(np.float64), self.x + y, U * (np.abs(self.x + y) + 18 * np.abs(y)), "residual")
        x = X.astype(np.float64)
        want = x / np.sqrt((x * x).mean(1, keepdims=True) + EPS) * self.w2
        near(N.astype(np.float64), want, 18 * U * np.abs(want), "norm")
        assert np.array_equal(self.XQ.download(np.uint8).reshape(self.rows, self.qx)[:rows, :HIDDEN // 32 * 40], orc.quant_q8(N))


@pytest.mark.parametrize("kind", (synth.KIND_Q4_0, synth.KIND_Q4_K))
def test_layer(dev, orc, kind):
    y = Layer(dev, kind, 170)
    # a prompt of 70 and the first 65 of another, packed, from zeros
    y.feed(135, [-1, -1], [3, 4], [0, 70, 135])
    y.run(135, 135, cu=y.cu)
    y.check([70, 65], orc)
    # the second one's next chunk alone
    y.feed(33, [3, 4], [3, 4], [0, 0, 33])
    y.run(33, 33, cu=y.cu)
    y.check([0, 33], orc)
    s = dev.Stream()
    # decode steps in place
    y.run(2, 1, decode=True, stream=s.s)  # the GEMVs' workspaces of this size, before the capture
    s.sync()
    graph = dev.Graph(s, lambda st: y.run(2, 1, decode=True, stream=st))
    for k in range(4):
        at = [3, 4] if k % 2 else [4, 3]
        y.feed(2, at, at)
        graph.launch()
        s.sync()
        y.check([1, 1], orc, decode=True)
    del graph
    # verify steps of three tokens, of which the first, second or third was the last accepted
    y.feed(6, [3, 4], [0, 1, 2, 5, 6, 7])
    y.run(6, 3, decode=True, each=1, stream=s.s)
    s.sync()
    graph = dev.Graph(s, lambda st: y.run(6, 3, decode=True, each=1, stream=st))
    at = [3, 4]
    for took in ((0, 2), (1, 1), (2, 0)):
        free = [i for i in range(SLOTS) if i not in at]
        to = free[:2] + [at[0]] + free[2:5]
        y.feed(6, at, to)
        graph.launch()
        s.sync()
        y.check([3, 3], orc, decode=True, each=True)
        at = [to[took[0]], to[3 + took[1]]]
    del graph
