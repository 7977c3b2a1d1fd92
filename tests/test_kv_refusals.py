"""What the cache operators refuse on the host, before any launch, on the CPU against the HIP runtime that does nothing
(capi/hip_stub.c)."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))

APPEND = dict(k=4096, v=4096, q=4096, qo=8192, qt=0, n_q=8, T=3, ks=512, vs=512, qs=512, qos=512, cu=None, freq=4096, n_rot=64, rope=1)
KV = dict(type=1, n_kv=2, hd=64, page=16, n_pages=9, k=4096, v=4096, n_seq=2, max_pages=40, pages=4096, len=4096)

BAD = {
    "append": [("kv", dict(type=0)), ("kv", dict(type=3)), ("kv", dict(n_kv=0)), ("kv", dict(n_kv=1025)), ("kv", dict(hd=96)), ("kv", dict(page=8)), ("kv", dict(page=48)),
               ("kv", dict(page=1 << 17)), ("kv", dict(n_pages=0)), ("kv", dict(n_pages=1 << 31)), ("kv", dict(k=None)), ("kv", dict(v=4104)), ("kv", dict(pages=None)), ("kv", dict(len=4098)),
               ("kv", dict(n_seq=0)), ("kv", dict(n_seq=(1 << 20) + 1)), ("kv", dict(max_pages=0)), ("kv", dict(max_pages=1 << 27)),
               (None, dict(n_q=0)), (None, dict(n_q=7)), (None, dict(n_q=2 * 129)), (None, dict(T=0)), (None, dict(T=1 << 22)), (None, dict(k=None)), (None, dict(v=None)),
               (None, dict(v=4097)), (None, dict(qo=None)), (None, dict(qt=2)), (None, dict(qo=8194)), (None, dict(ks=127)), (None, dict(vs=127)), (None, dict(qs=511)),
               (None, dict(qos=511)), (None, dict(rope=3)), (None, dict(rope=-1)), (None, dict(freq=None)), (None, dict(n_rot=0)), (None, dict(n_rot=7)), (None, dict(n_rot=66)),
               (None, dict(qo=4096, qos=513)), (None, dict(qo=4096, qt=1)), (None, dict(cu=4098)), (None, dict(cu=4096, T=(1 << 22) + 1))],
}
ATTN = dict(q=4096, y=8192, type=0, n_q=8, T=3, qs=512, ys=512, scale=0.125, ws=4096, ws_bytes=1 << 30, window=0, q8=None, q8s=0)
ATTN_BAD = [b for b in BAD["append"] if b[0] == "kv"] + [
    (None, c) for c in (dict(q=None), dict(y=None), dict(y=4096), dict(type=2), dict(type=3), dict(n_q=0), dict(n_q=7), dict(T=0), dict(qs=511), dict(ys=511), dict(q=4098), dict(y=8193),
                        dict(ws=None), dict(ws=4104), dict(ws_bytes=65536), dict(q8=12289, q8s=640), dict(q8=12288, q8s=636), dict(q8=12288, q8s=642),
                        dict(q8=4096, q8s=640), dict(q8=8192, q8s=640))]
BAD["decode"] = ATTN_BAD + [(None, dict(T=33)), (None, dict(n_q=256, T=2, qs=1 << 14, ys=1 << 14)), ("kv", dict(n_seq=1 << 20, n_kv=128)),
                             ("kv", dict(n_seq=33, max_pages=1 << 26))]
BAD["prefill"] = ATTN_BAD + [(None, dict(cu=4098)), (None, dict(T=1 << 22)), (None, dict(cu=4096, T=(1 << 22) + 1)), ("kv", dict(n_seq=1 << 20, n_kv=64))]
BASE = {"append": APPEND, "decode": ATTN, "prefill": ATTN}
GOOD = {
    "append": [{}, dict(q=None, qo=None, n_q=0, qs=0, qos=0), dict(cu=4096, T=100), dict(rope=0, freq=None, n_rot=0), dict(qt=1), dict(qo=4096), dict(n_q=256, qs=1 << 14, qos=1 << 14)],
    "decode": [{}, dict(type=1), dict(window=5), dict(y=None, q8=12288, q8s=640), dict(q8=12288, q8s=644), dict(T=32), dict(n_q=256, T=1, qs=1 << 14, ys=1 << 14)],
    "prefill": [{}, dict(type=1), dict(window=5), dict(cu=4096, T=5000), dict(y=None, q8=12288, q8s=640), dict(q8=12288, q8s=644), dict(T=4000), dict(n_q=256, T=1, qs=1 << 14, ys=1 << 14)],
}


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    d = tmp_path_factory.mktemp("hip")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-w", os.path.join(HERE, "capi", "hip_stub.c"), "-o", str(d / "libamdhip64.so.7")], check=True)
    return str(d)


def calls(stub, op, changes):
    """(error or '', launches, bytes of device memory asked for) of each call."""
    code = f"""
import sys; sys.path[:0] = {sys.path!r}
import ctypes as C, amdc
hip = C.CDLL("libamdhip64.so.7")
amdc.open_device()
n, l = C.c_size_t.in_dll(hip, "stub_bytes"), C.c_uint.in_dll(hip, "stub_launches")
f = {{"append": amdc.kv_append, "decode": getattr(amdc, "attn_decode", None), "prefill": getattr(amdc, "attn_prefill", None)}}[{op!r}]
for where, change in {changes!r}:
    kv, a = dict({KV!r}), dict({BASE[op]!r})
    (kv if where == "kv" else a).update(change)
    n.value = l.value = 0
    try:
        f(amdc.Kv(**kv), **a)
        e = ""
    except amdc.AmdcError as err:
        e = str(err)
    print(repr((e, l.value, n.value)))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=60, env=dict(os.environ, LD_LIBRARY_PATH=stub))
    assert r.returncode == 0, r.stderr[-800:]
    got = [eval(line) for line in r.stdout.splitlines()]
    assert len(got) == len(changes)
    return got


@pytest.mark.parametrize("op", sorted(BASE))
def test_refused(stub, op):
    for change, (err, launches, _) in zip(BAD[op], calls(stub, op, BAD[op])):
        assert err and launches == 0, change


@pytest.mark.parametrize("op", sorted(BASE))
def test_taken(stub, op):
    """One launch each (prompts: and one that joins, where few rows are split over the positions), and no allocation: every call can be
    captured."""
    for change, got in zip(GOOD[op], calls(stub, op, [(None, c) for c in GOOD[op]])):
        split = op == "prefill" and change.get("T", 3) < 4000
        assert got == ("", 2 if split else 1, 0), change


def test_kv_bytes():
    import amdc
    assert amdc.kv_bytes(1, 8, 128, 16, 10) == 8 * 128 * 16 * 10 * 2
    assert amdc.kv_bytes(2, 4, 256, 64, 3) == 4 * 256 * 64 * 3 * 2
    for bad in ((0, 8, 128, 16, 1), (1, 8, 80, 16, 1), (1, 8, 128, 24, 1), (1, 0, 128, 16, 1), (1, 8, 128, 16, 0), (1, 8, 64, 64, 1 << 27)):
        with pytest.raises(amdc.AmdcError):
            amdc.kv_bytes(*bad)
