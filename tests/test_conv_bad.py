"""What amdc_conv makes of slots that only the device sees: a sequence that starts from outside the pool is NaN in all of its
rows and no other is, and its slots stay."""
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
