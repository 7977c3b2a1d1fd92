"""What the operators of a linear-attention layer refuse on the host, before any launch, and that none allocates, on the CPU against the HIP
runtime that does nothing (capi/hip_stub.c)."""
import os
import subprocess
import sys

import pytest

from test_kv_refusals import stub  # noqa: F401 (the fixture)

SLOTS = dict(n_seq=2, n_slots=9, from_=4096, to=4096)
GDN = dict(n_k=2, n_v=4, dk=64, dv=48, order=0, scale=0.125, eps=1e-6, A=4096, dt=4096)
CONV = dict(states=4096, x=4096, w=4096, bias=4096, y=8192, type=0, ch=130, width=4, T=3, xs=130, ys=130, cu=None, each=0, act=1)
DECODE = dict(states=4096, q=4096, k=4096, v=4096, a=4096, b=4096, y=8192, type=0, T=3, qs=448, ks=448, vs=448, as_=4, bs=4, ys=192, each=0)
PREFILL = {**{k: v for k, v in DECODE.items() if k != "each"}, "cu": None, "ws": 4096, "ws_bytes": 1 << 40}
GATE = dict(x=4096, type=1, w=4096, z=8192, y=16384, n_h=3, hd=64, eps=1e-6, gate=0, q=32768, T=3, xs=384, zs=768, ys=768, qs=240)
RES = dict(x=4096, w1=4096, scale=1.0, res=8192, h=16384, w2=4096, y=32768, n=96, eps=1e-6, q=65536, T=3, xs=384, rs=384, hs=384, ys=384, qs=120)
BASE = {"conv": CONV, "gdn_decode": DECODE, "gdn_prefill": PREFILL, "norm_gate_q8": GATE, "norm_res_q8": RES}

SLOTS_BAD = [("slots", c) for c in (dict(n_seq=0), dict(n_seq=(1 << 20) + 1), dict(n_slots=0), dict(n_slots=1 << 31), dict(from_=None), dict(to=None), dict(from_=4098), dict(to=4097))] + [
    (None, c) for c in (dict(states=None), dict(states=4104), dict(T=0), dict(T=(1 << 21) + 1), dict(type=3), dict(type=-1))]
GDN_BAD = SLOTS_BAD + [("gdn", c) for c in (dict(n_k=0), dict(n_v=0), dict(n_v=5), dict(n_v=1026), dict(dk=32), dict(dk=96), dict(dk=256), dict(dv=0), dict(dv=40), dict(dv=272), dict(order=2),
                                             dict(order=-1), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(A=None), dict(dt=None), dict(A=4098), dict(dt=4097))] + [
    (None, c) for c in (dict(q=None), dict(k=None), dict(v=None), dict(a=None), dict(b=None), dict(y=None), dict(q=4098), dict(k=4097), dict(v=4098), dict(a=4098), dict(b=4098), dict(y=8194),
                        dict(y=4096), dict(type=1, k=4097), dict(qs=127), dict(ks=127), dict(vs=191), dict(as_=3), dict(bs=3), dict(ys=191))]
BAD = {
    "conv": SLOTS_BAD + [(None, c) for c in (dict(ch=0), dict(ch=(1 << 20) + 1), dict(width=1), dict(width=5), dict(x=None), dict(w=None), dict(y=None), dict(x=4098), dict(w=4097), dict(bias=4098),
                                             dict(y=8194), dict(y=4096), dict(act=2), dict(act=-1), dict(xs=129), dict(ys=129), dict(each=1, T=17), dict(each=1, cu=4096), dict(cu=4098),
                                             dict(cu=4096, T=(1 << 22) + 1), dict(T=1 << 21, ch=1 << 20, xs=1 << 20, ys=1 << 20))],
    "gdn_decode": GDN_BAD + [(None, dict(T=17)), (None, dict(T=17, each=1))],
    "gdn_prefill": GDN_BAD + [(None, c) for c in (dict(cu=4098), dict(cu=4096, T=(1 << 22) + 1), dict(ws=None), dict(ws=4104), dict(ws_bytes=15), dict(vs=1 << 23), dict(ys=1 << 23))],
    "norm_gate_q8": [(None, c) for c in (dict(x=None), dict(w=None), dict(z=None), dict(y=None, q=None), dict(T=0), dict(T=65536), dict(type=3), dict(gate=2), dict(gate=-1), dict(hd=16), dict(hd=96),
                                         dict(hd=512), dict(n_h=0), dict(n_h=4097), dict(x=4097), dict(w=4098), dict(z=8194), dict(y=16386), dict(q=32770), dict(xs=382), dict(xs=385), dict(zs=764),
                                         dict(zs=770), dict(ys=764), dict(ys=769), dict(qs=236), dict(qs=242))],
    "norm_res_q8": [(None, c) for c in (dict(x=None), dict(res=None), dict(h=None), dict(w2=None), dict(y=None, q=None), dict(n=0), dict(n=48), dict(n=32800), dict(T=0), dict(T=65536),
                                        dict(x=4098), dict(w1=4098), dict(res=8193), dict(h=16386), dict(w2=4097), dict(y=32769), dict(q=65538), dict(xs=380), dict(rs=380), dict(hs=380), dict(ys=380),
                                        dict(xs=386), dict(rs=386), dict(hs=386), dict(ys=386), dict(qs=116), dict(qs=122), dict(y=16384), dict(h=8192, hs=388), dict(h=4096, hs=388))],
}
GOOD = {
    "conv": [{}, dict(bias=None), dict(type=2), dict(each=1), dict(cu=4096, T=100), dict(act=0), dict(width=2), dict(T=16, each=1), dict(ch=1, xs=1, ys=1)],
    "gdn_decode": [{}, dict(type=1), dict(each=1), dict(T=16), dict(T=1)],
    "gdn_prefill": [{}, dict(type=2), dict(cu=4096, T=500), dict(T=1), dict(T=17)],
    "norm_gate_q8": [{}, dict(y=None), dict(q=None), dict(gate=1), dict(type=0, xs=768), dict(y=8192), dict(T=1, xs=0, zs=0, ys=0, qs=0)],
    "norm_res_q8": [{}, dict(w1=None), dict(y=None), dict(q=None), dict(h=8192), dict(h=4096), dict(T=1, xs=0, rs=0, hs=0, ys=0, qs=0), dict(n=32768, T=1)],
}


def calls(stub, op, changes):  # noqa: F811
    """(error or '', launches, bytes of device memory asked for) of each call."""
    code = f"""
import sys; sys.path[:0] = {sys.path!r}
import ctypes as C, amdc
nan = float("nan")
hip = C.CDLL("libamdhip64.so.7")
amdc.open_device()
n, l = C.c_size_t.in_dll(hip, "stub_bytes"), C.c_uint.in_dll(hip, "stub_launches")
for where, change in {changes!r}:
    sl, g, a = dict({SLOTS!r}), dict({GDN!r}), dict({BASE[op]!r})
    {{"slots": sl, "gdn": g}}.get(where, a).update(change)
    pre = [] if {op!r}.startswith("norm") else [amdc.Slots(**sl)]
    if {op!r}.startswith("gdn"):
        pre = [amdc.Gdn(**g)] + pre
    n.value = l.value = 0
    try:
        getattr(amdc, {op!r})(*pre, **a)
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
def test_refused(stub, op):  # noqa: F811
    for change, (err, launches, _) in zip(BAD[op], calls(stub, op, BAD[op])):
        assert err.startswith(op) and launches == 0, (change, err)


@pytest.mark.parametrize("op", sorted(BASE))
def test_taken(stub, op):  # noqa: F811
    """No allocation: every call can be captured."""
    for change, (err, launches, nbytes) in zip(GOOD[op], calls(stub, op, [(None, c) for c in GOOD[op]])):
        assert err == "" and nbytes == 0 and launches == (2 if op == "gdn_prefill" and {**PREFILL, **change}["T"] > 16 else 1), (change, err, launches)


def test_bytes():
    import amdc
    assert amdc.conv_bytes(10240, 4, 7) == 10240 * 3 * 7 * 4
    assert amdc.gdn_bytes(48, 128, 128, 5) == 48 * 128 * 128 * 5 * 4
    for bad in ((0, 4, 1), (8, 5, 1), (8, 1, 1), (8, 4, 0)):
        with pytest.raises(amdc.AmdcError):
            amdc.conv_bytes(*bad)
    for bad in ((0, 64, 64, 1), (4, 96, 64, 1), (4, 64, 72, 1), (4, 64, 64, 0), (4, 64, 272, 1)):
        with pytest.raises(amdc.AmdcError):
            amdc.gdn_bytes(*bad)
    for bad in (dict(n_k=3), dict(dk=32)):
        with pytest.raises(amdc.AmdcError):
            amdc.gdn_prefill_ws(amdc.Gdn(**{**GDN, **bad}), 1, 1)
    for n_seq, rows in ((0, 1), (1, 0), (1, (1 << 22) + 1), ((1 << 20) + 1, 5)):
        with pytest.raises(amdc.AmdcError):
            amdc.gdn_prefill_ws(amdc.Gdn(**GDN), n_seq, rows)


ALIASED = {"gdn_decode": [dict(a=8192), dict(b=8192)], "gdn_prefill": [dict(a=8192), dict(b=8192)],
           "norm_gate_q8": [dict(y=8192, ys=772), dict(y=8192, zs=772), dict(y=4096), dict(y=4096, type=0, xs=772), dict(y=4096, T=1)],
           "norm_res_q8": [dict(y=8192, ys=388), dict(y=4096, xs=388), dict(y=4096, h=4096)]}
IN_PLACE = {"norm_gate_q8": [dict(y=8192), dict(y=4096, type=0, xs=768), dict(y=8192, T=1, ys=0)], "norm_res_q8": [dict(y=8192), dict(y=4096), dict(y=8192, T=1, ys=0), dict(y=4096, h=8192)]}


@pytest.mark.parametrize("op", sorted(ALIASED))
def test_aliases(stub, op):  # noqa: F811
    """An output in an input's place is taken where a thread reads what it writes, and refused elsewhere."""
    for change, (err, launches, _) in zip(ALIASED[op], calls(stub, op, [(None, c) for c in ALIASED[op]])):
        assert err.startswith(op) and launches == 0, (change, err)
    if op in IN_PLACE:
        for change, (err, launches, _) in zip(IN_PLACE[op], calls(stub, op, [(None, c) for c in IN_PLACE[op]])):
            assert err == "" and launches == 1, (change, err)
