"""The kernels of a linear-attention layer in the built code object (amd.c_amd/amdc_kernels.hsaco): all that the host names are there, the
chunked delta rule on the matrix units, nothing in scratch memory, and as many waves on a SIMD as the kernels are laid out for."""
import os
import re

import pytest

from test_isa import HSACO, code  # noqa: F401 (code: the fixture)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
T = ("f32", "f16", "bf16")
CONV = [f"amdc_conv_w{w}_{t}{o}" for w in (2, 3, 4) for t in T for o in ("", "_odd")]
REC = [f"amdc_gdn_rec_h{h}_{t}" for h in (64, 128) for t in T]
PREP = [f"amdc_gdn_prep_h{h}_{t}" for h in (64, 128) for t in T]
SCAN = [f"amdc_gdn_scan_h{h}_{t}" for h in (64, 128) for t in T + ("f16_odd", "bf16_odd")]
NORM = [f"amdc_norm_gate_{t}" for t in T] + [f"amdc_norm_res_{c}" for c in (1, 2, 4, 8)]


def test_kernels(code):  # noqa: F811
    funcs, meta = code
    mine = {k for k in funcs if re.match(r"amdc_(conv|gdn|norm_gate|norm_res)_", k)}
    assert mine == set(CONV + REC + PREP + SCAN + NORM)
    for k in mine:
        assert any(mn.startswith("v_mfma_f32_16x16x32_f16") for _, mn, _ in funcs[k]) == (k in PREP + SCAN), k
        assert not any(mn.startswith("scratch_") for _, mn, _ in funcs[k]), k
        assert not any(mn.startswith("v_pk_") and mn.endswith("_f32") and mn[5:8] in ("add", "mul", "fma") for _, mn, _ in funcs[k]), k
        assert meta[k]["vgpr_count"] <= 256, "two waves on a SIMD"


@pytest.mark.parametrize("k", [k for k in CONV if not k.endswith("_odd")] + REC + PREP + NORM)
def test_wide_loads(code, k):  # noqa: F811
    """Rows of any alignment are read four values at a time."""
    assert any(mn in ("global_load_dwordx4", "global_load_dwordx2") for _, mn, _ in code[0][k])


def test_host_names():
    """Every kernel that the host resolves is in the code object, and these kernels once each."""
    host = open(os.path.join(ROOT, "amd.c_amd", "csrc", "amdc_host.c")).read()
    table = host[host.index("static const char *const kname[K_N] = {"):]
    table = table[:table.index("};")]
    names = []
    for macro, arg in re.findall(r'\b(KC|KT|KN)\("(\w+)"\)', table):
        names += [f"amdc_{arg}"] if macro == "KN" else [f"amdc_{arg}_{t}" for t in T] + ([f"amdc_{arg}_{t}_odd" for t in T] if macro == "KC" else [])
    blob = open(HSACO, "rb").read()
    mine = [n for n in names if re.match(r"amdc_(conv|gdn|norm_gate|norm_res)_", n)]
    assert sorted(mine) == sorted(CONV + REC + PREP + SCAN + NORM)
    assert all(n.encode() in blob for n in mine)
