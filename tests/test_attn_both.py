"""The same rows by amdc_attn_decode and by amdc_attn_prefill: five tokens of every sequence, on caches and queries of small whole numbers, so that the
scores' products and sums are exact and only what comes after them can differ."""
import numpy as np
import pytest

import test_attn_decode as dec
import test_attn_prefill as pre
from attncase import BF16, F16, F32, ULP, Case, attn64
from test_attn_nan import parts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ty,t,n_q,n_kv,hd", [(F16, F32, 24, 4, 256), (F16, F32, 6, 2, 64), (F16, F16, 28, 4, 128), (BF16, F32, 28, 4, 128), (BF16, BF16, 12, 2, 256), (F16, F32, 16, 2, 128)])
@pytest.mark.parametrize("window", (0, 150))
def test_five_rows(dev, ty, t, n_q, n_kv, hd, window):
    c = Case(dev, 640 + hd, ty, n_q, n_kv, hd, 16, (900, 333, 5, 4000), (5,) * 4)
    for k in c.k:
        k[:] = c.g.integers(-2, 3, k.shape)
    c.fill_all().upload()
    q, scale = c.g.integers(-2, 3, (20, n_q * hd)), 1.0 / np.sqrt(float(hd))
    d, p = (m.Call(c, t, *a, window=window, scale=scale, q=q, q8=True) for m, a in ((dec, (5,)), (pre, ())))
    yd, yp = d.launch().check(), p.launch().check()
    q8 = [parts(a.Q8.download(np.uint8).reshape(a.rows, a.q8s), a.w) for a in (d, p)]
    for b, L in enumerate(c.lens):
        k, v = c.stored(b)
        r = slice(5 * b, 5 * b + 5)
        want, av, _ = attn64(d.q[r], k, v, float(d.scale), np.arange(L - 5, L), window)
        top = max(np.abs(scale * (k[:, h // (n_q // n_kv)] @ d.q[r][:, h].T)).max() for h in range(n_q))
        assert top * 1.4427 < 16
        # an argument of the exponential is off by the rounding of a score under 16 (2^-21, in base 2), of the reference (2^-20) and of their
        # sum (2^-21), and where waves or parts join by as much as the first again: under 2.5 2^-20, a weight by 1.8 2^-20 with the
        # exponentials' 2^-22; in a 16-bit type by its half step as well; twice for the two sums; and this in either operator
        e = 2.0 ** -19 + (0 if t == F32 else ULP[t])
        tol = 4 * e * av + 2 * (L / 32 + 64) * 2.0 ** -24 * av
        assert (np.abs(yd[r] - yp[r]) <= tol + 2 * ULP[t] * np.abs(want)).all()
        # the scales of the Q8 copies, of the f32 results: the largest of a block, over 127
        big = tol.reshape(5, -1, 32).max(2)
        assert (np.abs(q8[0][1][r].astype(np.float64) - q8[1][1][r]) * 127 <= big * (1 + 2.0 ** -20) + 2.0 ** -21 * q8[0][1][r] * 127).all()
