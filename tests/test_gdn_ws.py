"""The size of amdc_gdn_prefill's workspace, as include/amdc_q4.h states it."""
import pytest

import amdc

HEADS = [(1, 1, 64, 16), (8, 16, 64, 64), (16, 48, 128, 128), (32, 128, 128, 16), (1, 1024, 64, 256), (1024, 1024, 128, 256)]
SIZES = [(1, 1), (1, 63), (1, 64), (1, 65), (1, 4000), (1, 1 << 22), (7, 7), (96, 96), (96, 5000), (1000, 40000), (1 << 20, 1 << 20), (1 << 20, 1 << 22)]


@pytest.mark.parametrize("n_k,n_v,dk,dv", HEADS)
def test_bound(n_k, n_v, dk, dv):
    g = amdc.Gdn(n_k, n_v, dk, dv, 0, 0.1, 1e-6, 4096, 4096)
    chunk, states = n_k * 768 * dk + n_v * 25600, 2 * 4 * n_v * dk * dv
    for n, rows in SIZES:
        got, chunks = amdc.gdn_prefill_ws(g, n, rows), rows // 64 + n
        chunks = min(chunks, (512 << 20) // chunk + 1)
        assert 0 <= got - chunk * chunks - states <= 16 * (chunks + 64) + 128
        assert chunk * chunks <= (512 << 20) + chunk
    for n, rows in SIZES:  # enough for all smaller ones
        assert all(amdc.gdn_prefill_ws(g, a, b) <= amdc.gdn_prefill_ws(g, n, rows) for a, b in SIZES if a <= n and b <= rows)
