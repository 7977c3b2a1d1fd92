"""Rows of a last sequence that go past T are reported by amdc_kv_check, also where they begin at T and no other workgroup has rows of
that sequence."""
import numpy as np
import pytest

import test_attn_prefill as pre
from attncase import F16, F32, Case, attn64
from test_attn_decode import bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_q,m,lens", [(4, 64, (70, 90)), (2, 128, (130, 90)), (4, 64, (3000, 90)), (4, 63, (70, 90)), (6, 64, (200, 90))])
def test_prompts(dev, n_q, m, lens):
    """T rows of G heads fill whole tiles of 128 rows (or, the last two, do not)."""
    c = Case(dev, 760 + m, F16, n_q, 2, 64, 16, lens, (m, 0), ragged=True).fill_all().upload()
    a = pre.Call(c, F32)
    c.dcu.upload(np.array([0, m, m + 5], np.int32))
    y = a.launch().got()
    k, v = c.stored(0)
    want, av, aq = attn64(a.q[:m], k, v, float(a.scale), np.arange(lens[0] - m, lens[0]), 0)
    assert (np.abs(y[:m] - want) <= bound(c, F32, want, av, aq, lens[0])).all()
    with pytest.raises(dev.AmdcError, match="rows outside"):
        dev.kv_check()
    dev.kv_check()
    c.dcu.upload(np.array([0, m, m], np.int32))
    a.launch().check()


@pytest.mark.parametrize("T,bad", [(64, (0, 64, 69)), (63, (0, 63, 2 ** 31 - 1)), (8, (0, 8, 9)), (64, (-1, 64, 64)), (64, (0, -5, -5))])
def test_append(dev, T, bad):
    c = Case(dev, 780, F16, 4, 2, 64, 16, (70, 90), (T, 0), ragged=True).upload()
    w = 2 * 64
    X = dev.DevBuf.of(np.ones((T, w), np.float32))
    c.dcu.upload(np.array(bad, np.int32))
    dev.kv_append(c.kv, X, X, None, None, F32, 0, T, w, w, cu=c.dcu)
    with pytest.raises(dev.AmdcError, match="rows outside"):
        dev.kv_check()
