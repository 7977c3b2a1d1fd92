"""amdc_attn_decode with more than 16 columns (T times the heads of a group) to a key / value head: the kernels on blocks of 32 columns, two
column tiles to a wave, their last block whole, half or a single column, and the same calls on heads of 256, in blocks of 16."""
import numpy as np
import pytest

from attncase import BF16, F16, F32, Case, as_float, attn64
from test_attn_decode import Call, bound
from test_attn_nan import parts, quantized

pytestmark = pytest.mark.gpu

CASES = [
    # type, t, n_q, n_kv, hd, T, window, lens
    (F16, F32, 28, 4, 128, 5, 0, (70, 3000)),
    (BF16, F32, 28, 4, 128, 8, 0, (3000, 8, 333)),
    (BF16, BF16, 24, 1, 64, 1, 0, (500, 31, 9000)),
    (BF16, BF16, 33, 1, 64, 2, 40, (500, 41)),
    (F16, F32, 17, 1, 128, 1, 0, (90, 0, 5000)),
    (F16, F16, 64, 2, 64, 1, 0, (90, 5000)),
    (BF16, F32, 11, 1, 64, 3, 5, (3, 4, 100, 2500)),
    (F16, F32, 20, 1, 256, 3, 0, (3, 700)),
]


def kernel(ty, t, hd, cols):
    return f"amdc_attn_dec_h{hd}_{ {F16: 'f16', BF16: 'bf16'}[ty]}" + ("_f32" if t == F32 else "") + ("_n2" if cols > 16 and hd <= 128 else "")


@pytest.mark.parametrize("i", range(len(CASES)))
def test_columns(dev, i):
    ty, t, n_q, n_kv, hd, T, window, lens = CASES[i]
    print(CASES[i], flush=True)
    c = Case(dev, 600 + i, ty, n_q, n_kv, hd, 16, lens, (T,) * len(lens)).fill_all().upload()
    a = Call(c, t, T, window).launch()
    assert dev.last_kernel() == kernel(ty, t, hd, T * n_q // n_kv)
    a.check()


GEOMETRIES = [(ty, t, hd) for ty in (F16, BF16) for t in (F32, ty) for hd in (64, 128)] + [(F16, F32, 256)]


@pytest.mark.parametrize("ty,t,hd", GEOMETRIES)
def test_infinities_where_rows_do_not_see(dev, ty, t, hd):
    """Three new tokens of 12 heads to a key / value head, so that both column tiles hold rows of two tokens: the second's and third's values
    infinite or NaN, the third's key too; the earlier rows' results are as if they were not there."""
    c = Case(dev, 610, ty, 24, 2, hd, 16, (45, 130, 2000), (3, 3, 3)).fill_all()
    for b, L in enumerate(c.lens):
        k, v = c.k[b].copy(), c.v[b].copy()
        v[L - 2, :, 5], v[L - 1, :, 7], k[L - 1, :, 3] = np.inf, np.nan, np.nan
        c.put(b, L - 2, L, k, v)
    c.upload()
    a = Call(c, t, 3).launch()
    got = a.got()
    for b, L in enumerate(c.lens):
        k, v = c.stored(b)
        q = a.q[3 * b:3 * b + 3]
        want, av, aq = attn64(q[:1], k, v, float(a.scale), [L - 3], 0)
        assert (np.abs(got[3 * b:3 * b + 1] - want) <= bound(c, t, want, av, aq, L)).all()
        mid = got[3 * b + 1]
        assert (mid[:, 5] == np.inf).all() if t != F32 else (~np.isfinite(mid[:, 5])).all()
        want, av, aq = attn64(q[1:2], k, np.where(np.isfinite(v), v, 0.0), float(a.scale), [L - 2], 0)
        keep = np.arange(hd) != 5
        assert (np.abs(mid - want[0]) <= bound(c, t, want, av, aq, L)[0])[:, keep].all()
        assert np.isnan(got[3 * b + 2]).all()


@pytest.mark.parametrize("ty,t,hd", GEOMETRIES)
def test_infinities_before_the_window(dev, ty, t, hd):
    c = Case(dev, 611, ty, 24, 2, hd, 16, (300, 90), (3, 3)).fill_all()
    for b, L in enumerate(c.lens):
        c.put(b, 0, L - 3 + 1 - 40, np.full_like(c.k[b], np.inf), np.full_like(c.v[b], np.nan))  # the first row sees 40 positions back
    c.upload()
    Call(c, t, 3, window=40).launch().check()


@pytest.mark.parametrize("ty,t,hd", GEOMETRIES)
def test_what_the_device_refuses(dev, ty, t, hd):
    for message, page, n in (("page outside", 999, None), ("length", None, 5000), ("length", None, 2)):
        c = Case(dev, 612, ty, 24, 2, hd, 16, (2000, 60), (3, 3)).fill_all()
        if page is not None:
            c.table[0, 70] = page
        c.upload()
        if n is not None:
            c.dlen.upload(np.array([n, 60], np.int32))
        a = Call(c, t, 3)
        y = a.launch().got()
        with pytest.raises(dev.AmdcError, match=message):
            dev.kv_check()
        assert np.isnan(y[:3]).all()
        k, v = c.stored(1)
        want, av, aq = attn64(a.q[3:], k, v, float(a.scale), [57, 58, 59], 0)
        assert (np.abs(y[3:] - want) <= bound(c, t, want, av, aq, 60)).all()
        assert not a.ws.download(np.uint32, 16384).any()


@pytest.mark.parametrize("ty,hd", [(F16, 64), (BF16, 64), (F16, 128), (BF16, 128), (F16, 256)])
def test_q8_copy(dev, ty, hd):
    c = Case(dev, 613, ty, 24, 2, hd, 16, (40, 0, 3000), (3, 3, 3)).fill_all().upload()
    a = Call(c, F32, 3, q8=True, pad=1)
    y = a.launch().check().astype(np.float32).reshape(a.rows, a.w)
    want = parts(quantized(dev, y), a.w)
    for again in range(2):
        got = a.Q8.download(np.uint8).reshape(a.rows, a.q8s)
        assert all(np.array_equal(g, x) for g, x in zip(parts(got, a.w), want))
        assert np.all(got[:, a.w // 32 * 40:] == 0xA5)
        a.Q8.fill(0xA5)
        a.Y = None
        a.launch()
        dev.sync()
