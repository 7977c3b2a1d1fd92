"""The cache and attention kernels in the built code object (amd.c_amd/amdc_kernels.hsaco): all that the host names are there, on the
matrix units; and what the loads into the LDS of the prompt kernels (inline assembly, out of the compiler's sight) rely on: m0 written
right before each and nowhere else, their buffer descriptors not from a vector instruction within five wait states (a hazard that the
compiler covers for its own loads), and one wait for all of them at the head of every tile."""
import os
import re

import pytest

from test_isa import HSACO, code, is_lds_dma, writes_m0  # noqa: F401 (code: the fixture)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = ("f16", "f16_f32", "bf16", "bf16_f32")
DEC = [f"amdc_attn_dec_h{h}_{t}" for h in (64, 128, 256) for t in TYPES] + [f"amdc_attn_dec_h{h}_{t}_n2" for h in (64, 128) for t in TYPES]
PRE = [f"amdc_attn_pre_h{h}_{t}" for h in (64, 128, 256) for t in TYPES]
OTHER = ["amdc_kv_append_f16", "amdc_kv_append_bf16"] + [f"amdc_attn_join_{t}" for t in ("f32", "f16", "bf16")]


def test_kernels(code):  # noqa: F811
    funcs, meta = code
    mine = {k for k in funcs if re.match(r"amdc_(kv|attn)_", k)}
    assert mine == set(DEC + PRE + OTHER)
    for k in DEC + PRE:
        assert any(mn.startswith("v_mfma_") for _, mn, _ in funcs[k]), k
        assert meta[k]["vgpr_count"] <= (512 if k == "amdc_attn_pre_h128_bf16_f32" else 256), "two waves on a SIMD"


def test_host_names():
    """Every kernel that the host resolves is in the code object, and these kernels once each."""
    host = open(os.path.join(ROOT, "amd.c_amd", "csrc", "amdc_host.c")).read()
    table = host[host.index("static const char *const kname[K_N] = {"):]
    table = table[:table.index("};")]
    names = []
    for macro, arg in re.findall(r"\b(KA2?|KN)\((\"\w+\")\)", table):
        arg = arg.strip('"')
        names += [f"amdc_{arg}"] if macro == "KN" else [f"amdc_{arg}_{t}" + ("_n2" if macro == "KA2" else "") for t in TYPES]
    blob = open(HSACO, "rb").read()
    assert all(n.encode() in blob for n in names)
    mine = [n for n in names if re.match(r"amdc_(kv|attn)_", n)]
    assert sorted(mine) == sorted(DEC + PRE + OTHER)


def _sgprs(ops):
    """The scalar registers named in an operand list."""
    regs = set()
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", ops):
        regs |= set(range(int(a), int(b) + 1))
    return regs | {int(a) for a in re.findall(r"\bs(\d+)\b", ops)}


@pytest.mark.parametrize("name", PRE)
def test_lds_loads(code, name):  # noqa: F811
    ins = code[0][name]
    loads = [i for i, (_, mn, ops) in enumerate(ins) if is_lds_dma(mn, ops)]
    assert len(loads) >= 8
    for i in loads:
        assert writes_m0(*ins[i - 2][1:]) and ins[i - 2][1] == "s_mov_b32" and ins[i - 1][1] == "s_nop", f"{ins[i][0]:#x}: not paired with its m0"
        need = _sgprs(ins[i][2].split(",", 1)[1])
        assert len(need) >= 4
        waits, j = 0, i - 1
        while waits < 5 and j >= 0:
            _, mn, ops = ins[j]
            if mn.startswith("v_read"):
                assert not need & _sgprs(ops.split(",", 1)[0]), f"{ins[i][0]:#x}: its descriptor is written by {mn} at {ins[j][0]:#x}, {waits} wait states before"
            waits += 1 + (int(ops.split()[0], 0) if mn == "s_nop" else 0)
            j -= 1
    assert sum(writes_m0(*x[1:]) for x in ins) == len(loads)
    # in both loops over tiles: those that every row sees, and the others
    marked = [ops for _, mn, ops in ins if mn == "s_waitcnt" and "expcnt(6)" in ops]
    assert len(marked) == 2 and all("vmcnt(0)" in ops for ops in marked), "the wait at the head of a tile"
