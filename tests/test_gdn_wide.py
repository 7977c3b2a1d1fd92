"""amdc_gdn_prefill where so many waves would have the sequences' heads that none goes token after token (sequences times value heads times
dv / 16 of 2^25 and more): also a sequence of one row goes through the chunks."""
import copy
import os
import subprocess
import sys

import numpy as np
import pytest

from attncase import F32, TINY
from lincase import U, Layer, Seqs, near, state_of

HERE = os.path.dirname(os.path.abspath(__file__))
N_SEQ, N_K, N_V, DK, DV = 2048, 1, 1024, 64, 256  # 2^25 waves
W = 2 * N_K * DK + N_V * DV


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    d = tmp_path_factory.mktemp("hip")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-w", os.path.join(HERE, "capi", "hip_stub_gdn.c"), "-o", str(d / "libamdhip64.so.7")], check=True)
    return str(d)


@pytest.mark.parametrize("strides", [(0, 0, 0, 0, 0, 0), (1, 1, 1, 1, 1, 1), (W, W, W, 2 * N_V, 2 * N_V, N_V * DV)])
def test_one_row_host(stub, strides):
    """A call of one row may have any strides; the kernels, which end their buffers behind whole rows, are given a row's width at least."""
    code = f"""
import sys; sys.path[:0] = {sys.path!r}
import ctypes as C, amdc
hip = C.CDLL("libamdhip64.so.7")
at = hip.stub_gdn_at
at.restype = C.c_size_t
amdc.open_device()
g = amdc.Gdn({N_K}, {N_V}, {DK}, {DV}, 0, 0.125, 1e-6, 4096, 4096)
qs, ks, vs, as_, bs, ys = {strides!r}
amdc.gdn_prefill(g, amdc.Slots({N_SEQ}, 3, 4096, 4096), 4096, 4096, 4096, 4096, 4096, 4096, 8192, 0, 1, qs, ks, vs, as_, bs, ys, 4096, 1 << 40, cu=4096)
print(*(at(i) for i in range(5)))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=60, env=dict(os.environ, LD_LIBRARY_PATH=stub))
    assert r.returncode == 0, r.stderr[-800:]
    vs, ys, few, tabs, packed = map(int, r.stdout.split())
    assert (few, packed) == (0, 1) and tabs > 0
    assert min(vs, ys) >= N_V * DV


def case(dev, seed, new, start, to, heads, strides=None):
    """The sequences of `new` (the others of 2048 have no row), checked on some heads."""
    g = np.random.default_rng(seed)
    s = Seqs(dev, seed, [new.get(b, 0) for b in range(N_SEQ)], start=[start.get(b, -1) for b in range(N_SEQ)], to=[to.get(b, -1) for b in range(N_SEQ)], ragged=True)
    s.n_slots = 2
    s.upload()
    L = Layer(g, s.rows, N_K, N_V, DK, DV).upload(dev)
    S = (0.3 * g.standard_normal((2, N_V, DV // 16, DK, 16))).astype(np.float32)
    dS, dy = dev.DevBuf.of(S), dev.DevBuf.of(np.full((s.rows, N_V * DV), 7, np.float32))
    ws = dev.DevBuf(dev.gdn_prefill_ws(L.gdn, N_SEQ, s.rows))
    ws.fill(0xFF)
    dev.gdn_prefill(L.gdn, s.slots, dS, *L.args(), dy, F32, s.T, *(strides or (*L.strides(), N_V * DV)), ws, ws.nbytes, cu=s.dcu)
    dev.kv_check()
    y = dy.download(np.float32).reshape(s.rows, N_V, DV)[:, heads]
    after = dS.download(np.float32).reshape(S.shape)
    c = copy.copy(L)  # the layer of those heads alone
    c.n_v, v = len(heads), L.x[:, 2 * DK:].reshape(s.rows, N_V, DV)[:, heads].reshape(s.rows, -1)
    c.x, c.ab = np.concatenate([L.x[:, :2 * DK], v], 1), L.ab[:, list(heads) + [N_V + h for h in heads]]
    c.A, c.dt = L.A[list(heads)], L.dt[list(heads)]
    kept = set(range(2))
    for b in new:
        old = state_of(S[start[b]])[heads] if start.get(b, -1) >= 0 else np.zeros((len(heads), DK, DV))
        want, err, st, es = c.run64(s.at(b), old, chunk=64)
        near(y[s.at(b)].astype(np.float64), want, err + U * np.abs(want) + TINY[F32], f"sequence {b}")
        if to.get(b, -1) >= 0:
            kept.discard(to[b])
            near(state_of(after[to[b]])[heads].astype(np.float64), st[-1], es[-1], f"state {b}")
    assert all(np.array_equal(after[i], S[i]) for i in kept)


@pytest.mark.gpu
@pytest.mark.parametrize("strides", (None, (0,) * 6, (1, 2, 3, 4, 5, 6)))
def test_one_row(dev, strides):
    case(dev, 1401, {1500: 1}, {1500: 1}, {1500: 0}, [0, 1, 517, 1023], strides)


@pytest.mark.gpu
def test_rows(dev):
    """Sequences of one, a few and more than a chunk's rows, far apart: in different launches."""
    case(dev, 1402, {0: 1, 7: 66, 700: 16, 2047: 3}, {7: 0, 2047: 1}, {7: 0, 2047: 1}, [2, 1000])


@pytest.mark.gpu
@pytest.mark.parametrize("at", (None, 10, 500, 1001, 1500, 2000))
def test_rows_outside(dev, at):
    """A sequence whose rows decrease is reported, wherever it stands: its chunks' numbers decrease too, by more than a launch takes."""
    rows = 1920
    L = Layer(np.random.default_rng(1403), 1, N_K, N_V, DK, DV).upload(dev)
    s = Seqs(dev, 1403, [0] * N_SEQ, start=[-1] * N_SEQ, to=[-1] * N_SEQ, ragged=True)
    s.cu[1:] = rows
    s.cu[at or N_SEQ:N_SEQ] = 0
    s.upload()
    x, ab, y, dS = dev.DevBuf(4 * rows * W), dev.DevBuf(4 * rows * 2 * N_V), dev.DevBuf(4 * rows * N_V * DV), dev.DevBuf(4)
    x.fill(0), ab.fill(0)
    ws = dev.DevBuf(dev.gdn_prefill_ws(L.gdn, N_SEQ, rows))
    dev.gdn_prefill(L.gdn, s.slots, dS, x.ptr, x.ptr + 4 * DK, x.ptr + 8 * DK, ab.ptr, ab.ptr + 4 * N_V, y, F32, rows, W, W, W, 2 * N_V, 2 * N_V, N_V * DV, ws, ws.nbytes, cu=s.dcu)
    if at:
        with pytest.raises(dev.AmdcError, match="rows outside"):
            dev.kv_check()
    dev.kv_check()
