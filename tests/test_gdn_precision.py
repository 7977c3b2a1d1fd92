"""The errors of amdc_gdn_prefill's chunks, which the bounds of test_gdn_prefill.py (worst cases, summed over the tokens) do not tell
from those of operands that have lost their low parts.

The criterion: against 64 bits, the root mean square error of y and of the state is at most 4 times that of the recurrence in f32 on the same
inputs. An operand of two f16 parts has 22 bits, f32 has 24: where the recurrence rounds an operand or a product, a chunk's product rounds
at most 2^2 times more coarsely, and it has fewer roundings than the tokens have one after the other. Without one low part an operand has 11 bits, and
y's error is 20 to 2000 times the recurrence's, whichever operand of whichever product it is: shown on the CPU, with the arithmetic of
gdnchunk.py.

And what include/amdc_q4.h states: of a column's errors, by its largest |v| and |S|, a root mean square of 2^-23, the largest 2^-20; 2^-125 besides; the
range of norms that sums have room for."""
import numpy as np
import pytest

from attncase import BF16, F16, F32, as_float
from gdnchunk import PRODUCTS, chunked, errors, recurrence
from lincase import Layer, state_of
from test_gdn_decode import Call

TIMES = 4  # of the recurrence's
RMS, MOST = 2.0 ** -23, 2.0 ** -20
CASES = [(dk, keep) for dk in (64, 128) for keep in (None, 0.5, 0.9, 0.99999)]
ONLY_Y = ("qk", "QS", "AU")


def plain(L, S):
    return errors(L, slice(0, len(L.x)), S, *recurrence(L, slice(0, len(L.x)), S)[:2])[0]


@pytest.mark.parametrize("dk,keep", CASES)
def test_criterion(dk, keep):
    """The chunks' arithmetic meets it, and does not without any one low part: y's error is over 4 times the limit, the state's over it too where
    the product goes into the state."""
    g = np.random.default_rng(1700)
    L = Layer(g, 330, 2, 4, dk, 48, keep=keep)
    S, sl = (0.3 * g.standard_normal((4, dk, 48))).astype(np.float32), slice(0, 330)
    limit = [TIMES * e for e in plain(L, S)]
    rms, most = errors(L, sl, S, *chunked(L, sl, S))
    assert rms[0] <= limit[0] and rms[1] <= limit[1] and max(rms) <= RMS and max(most) <= MOST
    for p in PRODUCTS:
        for side in ("left", "right"):
            rms, _ = errors(L, sl, S, *chunked(L, sl, S, (p, side)))
            assert rms[0] > 4 * limit[0], (p, side)
            if p not in ONLY_Y and not (p == "KS" and keep == 0.5):  # at the end of a chunk the state has forgotten what it was before
                assert rms[1] > limit[1], (p, side)


@pytest.mark.gpu
@pytest.mark.parametrize("t", (F32, F16, BF16))
@pytest.mark.parametrize("dk,keep", CASES)
def test_prompt(dev, dk, keep, t):
    """The kernel, on inputs of the same kind; y of 16 bits is rounded to those, so there the state alone."""
    c = Call(dev, 1701, (330,), 2, 4, dk, 48, keep=keep, t=t, prefill=True, scale=None if t == F32 else 2.0).upload().launch()
    s, L = c.s, c.L
    raw, pool = c.results()
    S = c.S[s.start[0]]
    after = state_of(pool.reshape(s.n_slots, 4, 3, dk, 16))[s.to[0]]
    rms, most = errors(L, s.at(0), S, as_float(raw, t).reshape(330, 4, 48), after)
    limit = [TIMES * e for e in plain(L, S)]
    for i in (0, 1) if t == F32 else (1,):
        assert rms[i] <= limit[i] and rms[i] <= RMS and most[i] <= MOST, (i, rms[i] / limit[i] * TIMES, np.log2(rms[i]), np.log2(most[i]))


@pytest.mark.gpu
@pytest.mark.parametrize("keep,amp", [(None, 0.3), (0.99999, 0.3), (1 - 1e-7, 0.3), (None, 1e4), (0.9, 1e-4)])
def test_long(dev, keep, amp):
    """4000 tokens: errors go on with the state, as f32's do."""
    c = Call(dev, 1702, (4000,), 1, 2, 128, 32, keep=keep, amp=amp, prefill=True).upload().launch()
    s, L = c.s, c.L
    raw, pool = c.results()
    S = c.S[s.start[0]]
    rms, most = errors(L, s.at(0), S, raw.reshape(4000, 2, 32).astype(np.float64), state_of(pool.reshape(s.n_slots, 2, 2, 128, 16))[s.to[0]])
    limit = [TIMES * e for e in plain(L, S)]
    assert rms[0] <= limit[0] and rms[1] <= limit[1] and max(rms) <= RMS and max(most) <= MOST, (np.log2(rms), np.log2(most), [r / l * TIMES for r, l in zip(rms, limit)])


@pytest.mark.gpu
@pytest.mark.parametrize("amp", (2.0 ** -100, 2.0 ** -110, 2.0 ** -118, 2.0 ** -126))
@pytest.mark.parametrize("dk", (64, 128))
def test_small(dev, dk, amp):
    """Values and states so small that the factor which takes a column back to its size is subnormal, off by 2^-150, and so is its product with
    the decay: each of two terms of y, of up to 2^23 times that factor, is off by 2 x 2^-127."""
    c = Call(dev, 1703, (200,), 2, 4, dk, 48, amp=amp, prefill=True)
    v = c.L.raw[:, 4 * dk:]
    v *= np.float32(amp)
    c.L.x = c.L.raw.astype(np.float64)
    s, L = c.upload().launch().s, c.L
    raw, pool = c.results()
    S = c.S[s.start[0]]
    want, last, sizes = recurrence(L, s.at(0), S, np.float64)
    most = np.maximum(sizes.max(0), np.abs(L.x[:, 4 * dk:]).max(0).reshape(4, 48))
    assert (np.abs(raw.reshape(200, 4, 48) - want) <= abs(float(L.scale)) * MOST * most + 2.0 ** -125).all()
    assert (np.abs(state_of(pool.reshape(s.n_slots, 4, 3, dk, 16))[s.to[0]] - last) <= MOST * most[:, None] + 2.0 ** -125).all()


@pytest.mark.gpu
@pytest.mark.parametrize("prefill", (False, True))
@pytest.mark.parametrize("dk", (64, 128))
def test_large(dev, dk, prefill):
    """Norms of keys and queries of up to 2^40, of values and of the state's columns up to 2^80."""
    c = Call(dev, 1704, (140, 70) if prefill else (16, 16), 2, 4, dk, 48, amp=2.0 ** 74, prefill=prefill)
    x = c.L.raw
    x[:, :4 * dk] *= np.float32(2.0 ** 35)
    x[:, 4 * dk:] *= np.float32(2.0 ** 72)
    c.L.x = x.astype(np.float64)
    n = np.linalg.norm(c.L.x[:, :4 * dk].reshape(len(x), 4, dk), axis=2).max()
    col = np.linalg.norm(c.S.astype(np.float64), axis=2).max()
    val = np.linalg.norm(c.L.x[:, 4 * dk:].reshape(len(x), 4, 48), axis=2).max()
    assert 2.0 ** 37 < n < 2.0 ** 40 and 2.0 ** 77 < col < 2.0 ** 80 and 2.0 ** 74 < val < 2.0 ** 80
    c.upload().launch().check()
