"""Packed batches of relative-position attention on the host: workspaces grow with the tokens and the sequences, not with their product, whatever the hint says."""
import ctypes as C

import pytest

from spokennlp_amd import lib as L


def _ws(T, B, hint, heads=12, kv_heads=12, D=64, span=128, dtype=0):
    c = L.RelposCfg(dtype=dtype, table_dtype=1, B=B, Lq=hint, Lk=hint, Tq=T, Tk=T, heads=heads, kv_heads=kv_heads, D=D, span=span, buckets=32, scale=0.125,
                    map=256, table=256, cu_q=256, cu_k=256)
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        getattr(c, n + "_stride")[:] = (0, heads * D, D)
    lib = L.load()
    assert lib.amdseg_relpos_attn_ws_bytes(C.byref(c), 0) == 0
    return lib.amdseg_relpos_attn_ws_bytes(C.byref(c), 1)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("T,B", [(1, 1), (64, 1), (18000, 24), (16384, 256), (32768, 256), (131072, 2048), (131072, 4096), (1 << 20, 64)])
def test_workspace_of_a_packed_batch(T, B, dtype):
    """per head and row: two floats; per head and row block (at least 64 rows, and at most one short one a sequence): the 2 (span + 112) + 1 sums over equal rel"""
    nd, heads = 2 * (128 + 112) + 1, 12
    most = 4 * heads * (2 * T + nd * (T // 64 + B + 1)) + 4096
    for hint in (1, 64, 300, T):
        n = _ws(T, B, hint, dtype=dtype)
        assert 0 < n <= most, (hint, n, most)
        assert n == _ws(T, B, 1, dtype=dtype), hint


def test_workspace_of_many_sequences_with_a_long_one():
    """256 sequences in 32 thousand tokens, no hint: some tens of MiB"""
    assert _ws(32768, 256, 32768) < 32 << 20
