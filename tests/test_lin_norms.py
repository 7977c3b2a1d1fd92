"""amdc_norm_gate_q8 and amdc_norm_res_q8 against their formulas in 64 bits; their Q8 copies are amdc_quant_q8's bits."""
import numpy as np
import pytest

from attncase import BF16, F16, F32
from lincase import U, near, sigmoid, typed

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.mark.parametrize("n_h,hd,T", [(48, 128, 1), (32, 128, 70), (1, 32, 1), (5, 64, 3), (3, 256, 9), (7, 32, 33), (33, 64, 2), (1, 256, 300)])
@pytest.mark.parametrize("t", (F32, F16, BF16))
@pytest.mark.parametrize("gate", (0, 1))
@pytest.mark.parametrize("pads", ((0, 0, 0), (4, 8, 4), (1, 3, 2)))
def test_gate(dev, orc, n_h, hd, T, t, gate, pads):
    g = np.random.default_rng(n_h * hd + T)
    n = n_h * hd
    xw, zw, yw = (n + p for p in pads)
    raw, x = typed(g.standard_normal((T, xw)) * 10.0 ** g.integers(-2, 3, (T, 1)), t)
    z = (4 * g.standard_normal((T, zw))).astype(np.float32)
    w = (1 + 0.3 * g.standard_normal(hd)).astype(np.float32)
    qs = n // 32 * 40 + 4 * pads[0]
    X, Z, W = dev.DevBuf.of(raw), dev.DevBuf.of(z), dev.DevBuf.of(w)
    Y, Q = dev.DevBuf.of(np.full((T, yw), 7, np.float32)), dev.DevBuf.of(np.full((T, qs), 7, np.uint8))
    dev.norm_gate_q8(X, t, W, Z, Y, n_h, hd, EPS, gate, Q, T, raw.itemsize * xw, 4 * zw, 4 * yw, qs)
    y = Y.download(np.float32).reshape(T, yw)
    xh, zz = x[:, :n].reshape(T, n_h, hd), z[:, :n].astype(np.float64)
    want = (xh / np.sqrt((xh * xh).mean(2, keepdims=True) + EPS) * w).reshape(T, n) * sigmoid(zz) * (1 if gate else zz)
    # squares, their sum (9 deep), quotient, eps, root, reciprocal: half of 13, 3; three products; the sigmoid's (4 + |z|)
    near(y[:, :n].astype(np.float64), want, U * (20 + 2 * np.abs(zz)) * np.abs(want) + 1e-37, "y")
    assert (y[:, n:] == 7).all()
    q = Q.download(np.uint8).reshape(T, qs)
    assert np.array_equal(q[:, :n // 32 * 40], orc.quant_q8(np.ascontiguousarray(y[:, :n]))) and (q[:, n // 32 * 40:] == 7).all()
    # y alone, the Q8 copy alone, and in the gate's place: the same bits
    Q2 = dev.DevBuf.of(np.full((T, qs), 7, np.uint8))
    dev.norm_gate_q8(X, t, W, Z, None, n_h, hd, EPS, gate, Q2, T, raw.itemsize * xw, 4 * zw, 0, qs)
    assert np.array_equal(Q2.download(np.uint8).reshape(T, qs), q)
    dev.norm_gate_q8(X, t, W, Z, Z, n_h, hd, EPS, gate, None, T, raw.itemsize * xw, 4 * zw, 4 * zw)
    assert np.array_equal(Z.download(np.float32).reshape(T, zw)[:, :n], y[:, :n])


def test_gate_far(dev):
    """Gates where exp(-z) overflows or vanishes; a head of zeros."""
    z = np.array([0, 1e-30, -1e-30, 88, -88, 100, -100, 1e4, -1e4, 3e38, -3e38] + [1.0] * 21, np.float32)
    x = np.ones((2, 32), np.float32)
    x[1] = 0
    X, Z, W, Y = dev.DevBuf.of(x), dev.DevBuf.of(np.stack([z, z])), dev.DevBuf.of(np.ones(32, np.float32)), dev.DevBuf(256)
    dev.norm_gate_q8(X, F32, W, Z, Y, 1, 32, EPS, 0, None, 2, 128, 128, 128)
    y = Y.download(np.float32).reshape(2, 32).astype(np.float64)
    want = z.astype(np.float64) * sigmoid(z)
    # the reciprocal gives 0 for a sigmoid under the smallest normal, 2^-126: that is from z = -87.3 to where exp(-z) overflows, at
    # -88.73, so that z times it is off by at most 89 2^-126
    near(y[0], want, U * (20 + 2 * np.abs(z.astype(np.float64))) * np.abs(want) + 5e-7 * np.abs(want) + 89 * 2.0 ** -126)
    assert (y[1] == 0).all()


@pytest.mark.parametrize("n,T", [(5120, 1), (32, 1), (64, 3), (4096, 2), (5120, 300), (992, 257), (8224, 5), (16384, 2), (17408, 256), (32768, 1), (32736, 260)])
@pytest.mark.parametrize("post", (True, False))
@pytest.mark.parametrize("pads", ((0, 0, 0, 0), (4, 8, 4, 4), (1, 2, 3, 5)))
def test_res(dev, orc, n, T, post, pads):
    g = np.random.default_rng(n + T)
    xw, rw, hw, yw = (n + p for p in pads)
    x, res = (3 * g.standard_normal((T, xw))).astype(np.float32), (20 * g.standard_normal((T, rw))).astype(np.float32)
    w1, w2 = ((1 + 0.3 * g.standard_normal(n)).astype(np.float32) for _ in range(2))
    scale = np.float32(0.22)
    qs = n // 32 * 40 + 4 * pads[0]
    X, R, W1, W2 = (dev.DevBuf.of(v) for v in (x, res, w1, w2))
    H, Y, Q = dev.DevBuf.of(np.full((T, hw), 7, np.float32)), dev.DevBuf.of(np.full((T, yw), 7, np.float32)), dev.DevBuf.of(np.full((T, qs), 7, np.uint8))
    dev.norm_res_q8(X, W1 if post else None, scale, R, H, W2, Y, n, EPS, Q, T, 4 * xw, 4 * rw, 4 * hw, 4 * yw, qs)
    h, y = H.download(np.float32).reshape(T, hw), Y.download(np.float32).reshape(T, yw)
    a, r = x[:, :n].astype(np.float64), res[:, :n].astype(np.float64)
    if post:
        a = a / np.sqrt((a * a).mean(1, keepdims=True) + EPS) * w1
    want = r + float(scale) * a
    # the mean square: 2 in a four, up to 8 fours, 6 + 4 to join, 2 more: half of 20; root, reciprocal, products; then one rounding
    eh = U * (np.abs(want) + 18 * float(scale) * np.abs(a))
    near(h[:, :n].astype(np.float64), want, eh, "h")
    hh = h[:, :n].astype(np.float64)  # from the h that it wrote
    want = hh / np.sqrt((hh * hh).mean(1, keepdims=True) + EPS) * w2
    near(y[:, :n].astype(np.float64), want, 18 * U * np.abs(want), "y")
    assert (h[:, n:] == 7).all() and (y[:, n:] == 7).all()
    q = Q.download(np.uint8).reshape(T, qs)
    assert np.array_equal(q[:, :n // 32 * 40], orc.quant_q8(np.ascontiguousarray(y[:, :n]))) and (q[:, n // 32 * 40:] == 7).all()
    # in the residual's place, the Q8 copy alone
    Q2 = dev.DevBuf.of(np.full((T, qs), 7, np.uint8))
    dev.norm_res_q8(X, W1 if post else None, scale, R, R, W2, None, n, EPS, Q2, T, 4 * xw, 4 * rw, 4 * rw, 0, qs)
    assert np.array_equal(R.download(np.float32).reshape(T, rw)[:, :n], h[:, :n]) and np.array_equal(Q2.download(np.uint8).reshape(T, qs), q)


def test_res_rows_alone(dev):
    """A row's bits do not depend on the rows beside it, within a number of rows that runs on the same threads."""
    g = np.random.default_rng(77)
    n = 5120
    x, res, w = (g.standard_normal((40, n)).astype(np.float32) for _ in range(3))
    X, R, W, H, Y = dev.DevBuf.of(x), dev.DevBuf.of(res), dev.DevBuf.of(w[0]), dev.DevBuf(40 * n * 4), dev.DevBuf(40 * n * 4)
    dev.norm_res_q8(X, W, 1.0, R, H, W, Y, n, EPS, None, 40, 4 * n, 4 * n, 4 * n, 4 * n)
    y = Y.download(np.uint32).reshape(40, n)
    dev.norm_res_q8(X.ptr + 17 * 4 * n, W, 1.0, R.ptr + 17 * 4 * n, H, W, Y, n, EPS)
    assert np.array_equal(Y.download(np.uint32, n), y[17])
