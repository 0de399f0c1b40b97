"""CPU half of the relative-position attention tests: the bucket scheme, the refusals (no kernel runs), the struct that crosses the C boundary."""
import ctypes as C
import math
import os
import re
import subprocess

import pytest
import torch

from spokennlp_amd import lib as L
from spokennlp_amd import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("nb,M,two", [(32, 128, True), (32, 128, False), (8, 48, True), (64, 512, True), (64, 200, False), (4, 7, True)])
def test_bucket_scheme(nb, M, two):
    got = ops.relpos_bucket_list(nb, M, two)
    assert len(got) == 2 * M + 1 and min(got) == 0 and max(got) == nb - 1 and got[M] == 0
    half = nb // 2 if two else nb
    m, steps = half // 2, half - half // 2
    for rel in range(-M, M + 1):
        n = abs(rel) if two else max(-rel, 0)
        if n < m:
            want = n
        else:
            x = m + math.log(n / m) / math.log(M / m) * steps
            if abs(x - round(x)) < 1e-9:                     # an edge: whole-number arithmetic decides, and it belongs to the bucket that begins there
                x = round(x)
            want = min(half - 1, math.floor(x))
        assert got[M + rel] == want + (half if two and rel > 0 else 0), rel


def test_bucket_scheme_refuses():
    for nb, M, two in ((3, 128, True), (1, 128, False), (32, 8, True), (0, 4, True)):
        with pytest.raises(ValueError):
            ops.relpos_bucket_list(nb, M, two)


def test_struct_layout(tmp_path):
    fields = [f for f, _ in L.RelposCfg._fields_]
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "amdseg.h"\nint main(void){printf("%zu\\n", sizeof(struct amdseg_relpos_cfg));\n' +
                   "".join(f'printf("%zu\\n", offsetof(struct amdseg_relpos_cfg, {f}));\n' for f in fields) + "return 0;}\n")
    exe = tmp_path / "p"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(L.RelposCfg)] + [getattr(L.RelposCfg, f).offset for f in fields]


def _cfg(**kw):
    """a configuration whose pointers are host addresses that are never followed: every call below is refused before a launch"""
    buf = (C.c_char * 65536)()
    p = (C.addressof(buf) + 255) // 256 * 256
    c = L.RelposCfg(dtype=0, table_dtype=1, B=2, Lq=8, Lk=8, heads=4, kv_heads=2, D=64, span=16, buckets=8, scale=0.125, map=p, table=p)
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        getattr(c, n + "_stride")[:] = (8 * 256, 256, 64)
    for n, x in kw.items():
        if n.endswith("_stride") and n != "mask_stride":
            getattr(c, n)[:] = x
        else:
            setattr(c, n, x)
    return c, p, buf


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(table_dtype=5), dict(kv_heads=3), dict(kv_heads=0), dict(heads=0), dict(D=12), dict(D=136), dict(D=0), dict(span=1025),
                                dict(span=-1), dict(buckets=0), dict(scale=0.0), dict(scale=float("nan")), dict(scale=-1.0), dict(B=-1), dict(Lq=-1), dict(Lk=(1 << 30) + 1),
                                dict(map=None), dict(table=None), dict(cu_q=256), dict(cu_q=256, cu_k=256, k_lens=256), dict(q_stride=(2048, 256, 60)),
                                dict(k_stride=(2048, 252, 64)), dict(out_stride=(2047, 256, 64))])
def test_c_entry_refuses(kw):
    c, p, _keep = _cfg(**kw)
    lib = L.load()
    assert lib.amdseg_relpos_attn_fwd(C.byref(c), p, p, p, p, None, None, 0, None) in (1001, 1002)
    assert lib.amdseg_relpos_attn_bwd(C.byref(c), p, p, p, p, p, p, p, p, p, p, p, 1 << 30, None) in (1001, 1002)


def test_c_entry_refuses_pointers_and_workspaces():
    c, p, _keep = _cfg()
    lib = L.load()
    assert lib.amdseg_relpos_attn_fwd(None, p, p, p, p, None, None, 0, None) == 1002
    for bad in (None, p + 8):
        assert lib.amdseg_relpos_attn_fwd(C.byref(c), bad, p, p, p, None, None, 0, None) == 1002
        assert lib.amdseg_relpos_attn_fwd(C.byref(c), p, p, p, bad, None, None, 0, None) == 1002
    n = lib.amdseg_relpos_attn_ws_bytes(C.byref(c), 1)
    assert n > 0
    assert lib.amdseg_relpos_attn_bwd(C.byref(c), p, p, p, p, p, p, p, p, p, p, p, n - 1, None) == 1002
    assert lib.amdseg_relpos_attn_bwd(C.byref(c), p, p, p, p, p, p, p, p, p, p, None, n, None) == 1002
    assert lib.amdseg_relpos_attn_bwd(C.byref(c), p, p, p, p, p, None, p, p, p, p, p, n, None) == 1002
    few, _, _k2 = _cfg(Lq=1, Lk=5000)
    n = lib.amdseg_relpos_attn_ws_bytes(C.byref(few), 0)
    assert n > 0 and lib.amdseg_relpos_attn_fwd(C.byref(few), p, p, p, p, None, p, n - 1, None) == 1002
    assert lib.amdseg_relpos_bias_fwd(p, 1, p, 16, 8, 4, 5, 5, 0, p + 4, 0, None) == 1002
    assert lib.amdseg_relpos_bias_fwd(p, 1, p, 16, 8, 4, 5, 5, 0, p, 3, None) == 1002
    assert lib.amdseg_relpos_bias_bwd(p, 0, p, 16, 8, 1, 4, 5, 5, 0, p, p, 8, None) == 1002
    assert lib.amdseg_relpos_bias_bwd(p, 0, p, 2000, 8, 1, 4, 5, 5, 0, p, p, 1 << 20, None) == 1002


def test_python_surface_refuses():
    q = torch.zeros(2, 8, 4, 64)
    with pytest.raises(ValueError, match="one GPU"):
        ops.relpos_attn_fwd(q, q, q, torch.zeros(8, 4), torch.zeros(17, dtype=torch.int32))
    with pytest.raises(ValueError, match="come together"):
        ops.relpos_attn_fwd(q, q, q, torch.zeros(8, 4), torch.zeros(17, dtype=torch.int32), cu_q=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        ops.relpos_bias_fwd(torch.zeros(8, 4), torch.zeros(17, dtype=torch.int32), 4, 4)
    with pytest.raises(ValueError):
        ops.relpos_bias_bwd(torch.zeros(1, 4, 4, 4), torch.zeros(17, dtype=torch.int32), 8)


def test_module_shapes_and_refusals():
    from spokennlp_amd import relpos as R
    m = R.RelPosSelfAttention(256, 4, kv_heads=2, buckets=16, max_distance=64)
    assert m.qkv.weight.shape == (512, 256) and m.table.shape == (16, 4) and m.bucket_map.tolist() == ops.relpos_bucket_list(16, 64, True)
    assert "bucket_map" not in m.state_dict()
    with pytest.raises(ValueError):
        R.RelPosSelfAttention(256, 4, kv_heads=3)
    with pytest.raises(ValueError):
        R.RelPosSelfAttention(256, 4, table=torch.nn.Parameter(torch.zeros(8, 4)))
    with pytest.raises(ValueError, match="columns"):
        R.relpos_self_attention(torch.zeros(1, 4, 500), 4, m.table, m.bucket_map)
    with pytest.raises(ValueError, match="one GPU"):
        m(torch.zeros(1, 4, 256))
