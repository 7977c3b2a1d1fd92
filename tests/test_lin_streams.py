"""The operators of a linear-attention layer on two streams at a time, each call with its own slots and workspace; a captured prompt
and an eager one that share a workspace, one after the other; and what the chain recorder does with them."""
import numpy as np
import pytest

from attncase import BF16, F32
from lincase import pool_of
from test_conv import Call as Conv
from test_gdn_decode import Call as Gdn

pytestmark = pytest.mark.gpu


def test_two_streams(dev):
    """Calls of one kind and of different kinds, whose launches overlap."""
    both = [(Gdn(dev, 1301 + i, (260, 70 + i), 2, 6, 128, 64, tiled=True, t=t, prefill=True).upload(), Gdn(dev, 1311 + i, (3,) * 40, 2, 4, 64, 64, each=True).upload(),
             Conv(dev, 1321 + i, (90, 1, 300 + i), 512, t=t).upload()) for i, t in enumerate((F32, BF16))]
    streams = dev.Stream(), dev.Stream()
    dev.sync()
    for rep in range(4):
        for s, cs in zip(streams, both):
            for c in cs:
                c.launch(s.s)
    for s in streams:
        s.sync()
    for cs in both:
        for c in cs:
            c.check()


def test_shared_workspace(dev):
    """Of a graph and of an eager call in the same stream: nothing is left in it that the next call needs."""
    a, b = Gdn(dev, 1331, (200, 64), 2, 4, 128, 128, prefill=True).upload(), Gdn(dev, 1332, (65, 3, 130), 1, 4, 64, 48, t=BF16, prefill=True).upload()
    b.ws = a.ws = a.ws if a.ws.nbytes > b.ws.nbytes else b.ws
    s = dev.Stream()
    graph = dev.Graph(s, lambda st: a.launch(st))
    for _ in range(3):
        for c in (a, b):
            c.dS.upload(pool_of(c.S)), c.dy.upload(c.y0)
        dev.sync()
        graph.launch()
        b.launch(s.s)
        graph.launch()
        s.sync()
        a.check(), b.check()
    del graph


def test_recorder(dev):
    """None of them can be recorded: the call fails, nothing runs, and so does the recording."""
    c, d, p = Conv(dev, 1341, (2, 2), 64).upload(), Gdn(dev, 1342, (2, 2)).upload(), Gdn(dev, 1343, (70, 3), prefill=True).upload()
    x, q = dev.DevBuf.of(np.ones((2, 64), np.float32)), dev.DevBuf.of(np.full((2, 80), 7, np.uint8))
    s = dev.Stream()
    for call in (lambda: c.launch(s.s), lambda: d.launch(s.s), lambda: p.launch(s.s), lambda: dev.norm_gate_q8(x, F32, x, x, None, 2, 32, 1e-6, 0, q, 2, 256, 256, 0, 80, stream=s.s),
                 lambda: dev.norm_res_q8(x, None, 1.0, x, x, x, None, 64, 1e-6, q, 2, 256, 256, 256, 0, 80, stream=s.s)):
        with pytest.raises(dev.AmdcError):
            with dev.ChainRecorder(s):
                with pytest.raises(dev.AmdcError):
                    call()
        s.sync()
    for k in (c, d, p):
        assert (k.dy.download(k.y0.dtype) == 7).all()
    assert (q.download(np.uint8) == 7).all() and (x.download(np.float32) == 1).all()
