"""Sequences as long as a table can say, 2^31 - 16 positions: the parts that a prompt tile's positions are split into cover them all, and both
attention operators read the last ones. The table repeats one page of 16 positions, but for its last entry."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from attncase import F16, F32, as_float, to16

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "amd.c_amd", "csrc")


def test_parts(tmp_path):
    src = tmp_path / "parts.c"
    src.write_text('#include "amdc_layout.h"\nuint32_t at(uint32_t n, uint32_t i, uint32_t p) { return amdc_part_at(n, i, p); }\n')
    subprocess.run(["gcc", "-std=c11", "-O2", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(tmp_path / "parts.so")], check=True)
    at = C.CDLL(str(tmp_path / "parts.so")).at
    at.restype, at.argtypes = C.c_uint32, [C.c_uint32] * 3
    for n in (1, 4, 5, 63, 64, 375, 9001, (1 << 25) - 1, 1 << 25, (1 << 26) - 1, 1 << 26):
        for parts in (1, 2, 3, 5, 32, 63, 64):
            assert [at(n, i, parts) for i in range(parts + 1)] == [n * i // parts for i in range(parts + 1)], (n, parts)


@pytest.mark.gpu
@pytest.mark.parametrize("t,hd", [(F16, 256), (F32, 128)])
def test_last_positions(dev, t, hd):
    """Of zero keys but for one of score 60 among the last 16: its value, e^60 times the weight of all the others."""
    entries = (1 << 27) - 1
    g = np.random.default_rng(790)
    K, V = np.zeros((2, 1, 1, hd // 8, 16, 8), np.uint16), to16(g.standard_normal((2, 1, 2, hd, 8)), F16)
    K[1, 0, 0, :, 5] = to16(np.full((hd // 8, 8), 60 * 16 / hd), F16)
    table = np.zeros(entries, np.int32)
    table[-1] = 1
    dK, dV, dT, dL = dev.DevBuf.of(K), dev.DevBuf.of(V), dev.DevBuf.of(table), dev.DevBuf.of(np.array([16 * entries], np.int32))
    kv = dev.Kv(F16, 1, hd, 16, 2, dK, dV, 1, entries, dT, dL)
    q = np.ones(hd, np.float32)
    Q, Y = dev.DevBuf.of(q if t == F32 else to16(q, t)), dev.DevBuf(hd * (4 if t == F32 else 2))
    want = as_float(V[1, 0, 0, :, 5], F16)
    for op in ("prefill", "decode"):
        size = dev.attn_prefill_ws(kv, 1, 1) if op == "prefill" else dev.attn_decode_ws(kv, 1, 1)
        ws = dev.DevBuf(size)
        ws.fill(0)
        Y.fill(0)
        print(op, flush=True)
        (dev.attn_prefill if op == "prefill" else dev.attn_decode)(kv, Q, Y, t, 1, 1, hd, hd, 1 / 16, ws, size)
        dev.sync()
        y = as_float(Y.download(np.float32 if t == F32 else np.uint16), t)
        # the one weight's parts, sum and division: a few roundings; the others' weights together 2^31 e^-60
        assert (np.abs(y - want) <= (4 * 2.0 ** -24 + (2.0 ** -11 if t == F16 else 0.0)) * np.abs(want) + 2.0 ** -50).all(), op
        dev.kv_check()
    for b in (dK, dV, dT, dL):
        b.free()
