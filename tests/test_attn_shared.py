"""What the host and the attention kernels both have to know is written once, in amdc_layout.h: neither of the two defines a constant under a
name that the other defines, nor a struct of kernel arguments of its own."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "amd.c_amd", "csrc")


def read(f):
    return open(os.path.join(CSRC, f)).read()


def test_written_once():
    host, attn, layout = (read(f) for f in ("amdc_host.c", "amdc_attn.h", "amdc_layout.h"))
    host = host[host.index("attention over a paged cache"):]
    host = host[:host.index("int amdc_probe_read")]
    names = [set(re.findall(r"^#define (\w+)", s, re.M)) for s in (host, attn)]
    assert not names[0] & names[1]
    for s in (host, attn):
        assert not re.search(r"^(typedef )?struct \w*[aA]rgs|^\} \w*args;", s, re.M)
        for shared in ("AMDC_ATTN_CNT", "AMDC_PRE_BM", "AMDC_PRE_MINTILES", "AMDC_PRE_MAXPARTS", "AMDC_PRE_W", "AMDC_PRE_BN", "AMDC_DEC_NW", "amdc_append_args", "amdc_attn_args"):
            assert re.search(rf"\b{shared}\b", s) and re.search(rf"\b{shared}\b", layout), shared
