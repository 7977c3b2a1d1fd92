"""amdc_kv_check loses no report, on the CPU against a HIP runtime that does nothing but keep the flag (capi/hip_stub_flag.c): one that
arrives between its look at the flag and its end is there for the next check."""
import os
import subprocess
import sys

import pytest

import test_attn_decode as dec
from attncase import F16, F32, Case

HERE = os.path.dirname(os.path.abspath(__file__))


def test_a_report_that_comes_late(tmp_path):
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-w", os.path.join(HERE, "capi", "hip_stub_flag.c"), "-o", str(tmp_path / "libamdhip64.so.7")], check=True)
    code = f"""
import sys; sys.path[:0] = {sys.path!r}
import ctypes as C, amdc
hip = C.CDLL("libamdhip64.so.7")
amdc.open_device()
late = C.c_uint.in_dll(hip, "stub_late")
def check():
    try:
        amdc.kv_check()
        print("-")
    except amdc.AmdcError as e:
        print(str(e).split(" met ")[1].split()[1])
check()
hip.stub_report(1)
late.value = 2
check(), check(), check()
late.value = 3
check(), check(), check()
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=60, env=dict(os.environ, LD_LIBRARY_PATH=str(tmp_path)))
    assert r.returncode == 0, r.stderr[-800:]
    assert r.stdout.split() == ["-", "page", "length", "-", "-", "outside", "-"]


@pytest.mark.gpu
def test_on_the_device(dev):
    """Each bad call is reported once; amdc_last_kernel stays the operator's."""
    c = Case(dev, 795, F16, 4, 2, 64, 16, (60,), (1,)).fill_all()
    c.table[0, 1] = 99
    c.upload()
    for _ in range(3):
        dec.Call(c, F32, 1).launch()
        with pytest.raises(dev.AmdcError, match="page outside"):
            dev.kv_check()
        assert dev.last_kernel() == "amdc_attn_dec_h64_f16_f32"
        dev.kv_check()
