"""What amdc_conv makes of slots and rows that only the device sees: a sequence that starts from outside the pool is NaN in all of its
rows and no other is, and its slots stay; of a sequence with rows outside 0 .. T none is written."""
import numpy as np
import pytest

from attncase import BF16, F16, F32, as_float
from test_conv import Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", (0, 1))
@pytest.mark.parametrize("ch,width,t", [(36, 4, F32), (36, 2, BF16), (77, 3, F16)])
@pytest.mark.parametrize("new,each", [((3, 40, 5), False), ((8, 9, 100), False), ((5, 5, 5), True), ((1, 1, 1), False)])
def test_start_outside(dev, new, each, ch, width, t, act):
    for lost, bad in ((0, -2), (1, 1 << 30), (2, None)):
        c = Call(dev, 1501 + lost, new, ch, width, t, act=act, each=each, bias=lost != 1)
        s = c.s
        s.start[lost] = s.n_slots if bad is None else bad
        c.upload().launch()
        with pytest.raises(dev.AmdcError, match="slot outside"):
            dev.kv_check()
        y = as_float(c.dy.download(c.y0.dtype).reshape(c.y0.shape), t)
        want = np.zeros(y.shape, bool)
        want[s.at(lost)] = True
        assert np.array_equal(np.isnan(y), want)
        pool = c.dpool.download(np.float32).reshape(c.pool.shape)
        mine = s.to[s.at(lost)] if each else s.to[[lost]]
        assert np.array_equal(pool[mine], c.pool[mine])
        others = [i for i in s.to if i not in mine]
        assert (pool[others] != c.pool[others]).any(axis=(1, 2)).all()


@pytest.mark.parametrize("cu", [(0, 40, 20, 48), (0, 48, 47, 48), (0, 3, 2, 48), (-1, 3, 43, 48), (0, 3, 43, 52), (-9, -9, 0, 48), (0, 48, 48, 47), (48, 40, 30, 20), (1 << 30, 48, 48, 48),
                                (0, 0, -(1 << 31), 48), (5, 5, 5, 5), (48, 48, 48, 48)])
def test_rows_outside(dev, cu):
    """Reported, wherever cu decreases or leaves 0 .. T; and no row that only such sequences name is written."""
    c = Call(dev, 1511, (3, 40, 5), 36, ragged=True).upload()
    c.s.dcu.upload(np.array(cu, np.int32))
    c.launch()
    good, fine = np.zeros(c.s.total, bool), True
    for a, b in zip(cu, cu[1:]):
        if 0 <= a <= b <= c.s.T:
            good[a:b] = True
        else:
            fine = False
    if fine:
        dev.kv_check()
    else:
        with pytest.raises(dev.AmdcError, match="rows outside"):
            dev.kv_check()
    dev.kv_check()
    assert (c.dy.download(np.float32).reshape(c.y0.shape)[~good] == 7).all()
