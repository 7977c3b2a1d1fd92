"""A scale that is not finite gives NaN in every row that takes part, in both attention operators."""
import numpy as np
import pytest

import test_attn_decode as dec
import test_attn_prefill as pre
from attncase import BF16, F16, F32, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ty,t,hd", [(F16, F16, 64), (F16, F32, 128), (BF16, BF16, 128), (BF16, F32, 256)])
@pytest.mark.parametrize("lens", [(90, 0, 40), (3000, 0, 40)])
@pytest.mark.parametrize("scale", (np.nan, np.inf, -np.inf))
def test_nan(dev, ty, t, hd, lens, scale):
    c = Case(dev, 740 + hd, ty, 4, 2, hd, 16, lens, (3, 3, 3)).fill_all().upload()
    for a in (dec.Call(c, t, 3, scale=scale), pre.Call(c, t, scale=scale), pre.Call(c, t, scale=scale, window=50)):
        y = a.launch().got()
        assert np.isnan(y[:3]).all() and np.isnan(y[6:]).all() and (y[3:6] == 0).all()
        dev.kv_check()
