"""Attention under a learned relative position bias (spokennlp_amd.ops.relpos_*) on a real MI355X against plain implementations in 64 bits.

Tolerances, from the arithmetic (u = half a step of the type: bf16 2^-8, fp32 2^-24; errors are 2-norms over a whole output, relative to its 2-norm):
 * bf16: an output is rounded once, the probabilities (forward) or p and ds (backward) once before their product, and delta inherits the rounding of `out`.
   Each is at most u per element; as independent errors uniform in a half step they have rms <= u / sqrt 3 times a factor between 1 / 2 and 1 (where the
   value stands in its binade).  Four of them in quadrature stay under 2 u / sqrt 3 = 4.6e-3; 2 u = 7.8e-3 is the bound used, and it is the sum bound for two
   roundings that all go the same way.
 * fp32: products accumulate at most 128 + 8192 terms, exp2 and the score's sum err by a few u times the score's size (|s| <= 40 here): 2e-5 = 335 u.
 * lse (fp32 from either type): scores are exact products summed in fp32, so abs error <= a few u times (|s| + 40): 2e-5 relative to max(1, |lse|).
 * the dense bias is one rounding of a table entry: fp32 exact, bf16 equal to torch's own rounding; its gradient is an fp32 sum taken as a tree: 2e-5."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64
TOL = {torch.bfloat16: 2 * 2.0 ** -8, torch.float32: 2e-5}


def _ops():
    from spokennlp_amd import ops
    return ops


def rel(a, b):
    a, b = a.to(F64), b.to(F64)
    n = float(b.norm())
    return float((a - b).norm()) / n if n else float((a - b).norm())


def ref_attention(q, k, v, table, lut, scale, seen, off, dout=None):
    """one sequence: q [Lq, H, D], k / v [Lk, Hk, D], seen bool [Lk] -> out, lse, gradients; 64 bits"""
    H, Hk, span = q.shape[1], k.shape[1], lut.numel() // 2
    req = dout is not None
    q, k, v, table = (x.detach().to(F64).requires_grad_(req) for x in (q, k, v, table))
    Lq, Lk = q.shape[0], k.shape[0]
    r = torch.arange(Lk, device=q.device)[None] - (torch.arange(Lq, device=q.device)[:, None] + off[0])
    bias = table[lut.long()[r.clamp(-span, span) + span]].permute(2, 0, 1)
    # rows of hidden keys may hold anything
    kk = torch.where(seen[:, None, None], k, torch.zeros_like(k)).repeat_interleave(H // Hk, 1)
    vv = torch.where(seen[:, None, None], v, torch.zeros_like(v)).repeat_interleave(H // Hk, 1)
    s = torch.einsum("ihd,jhd->hij", q, kk) * scale + bias
    vis = seen[None, :].expand(Lq, Lk)
    if off[1]:
        vis = vis & (r <= 0)
    s = s.masked_fill(~vis[None], -math.inf)
    blind = ~vis.any(1)
    p = torch.softmax(s.masked_fill(blind[None, :, None], 0.0), -1) * (~blind)[None, :, None]
    out = torch.einsum("hij,jhd->ihd", p, vv)
    lse = torch.logsumexp(s, -1) if Lk else torch.full((H, Lq), -math.inf, dtype=F64, device=q.device)
    if not req:
        return out, lse
    g = torch.autograd.grad(out, (q, k, v, table), dout.to(F64), allow_unused=True)
    return out, lse, [torch.zeros_like(x) if y is None else y for x, y in zip((q, k, v, table), g)]


def make(dev, dtype, B, Lq, Lk, H, Hk, D, buckets=32, max_distance=128, bidirectional=True, seed=0, fused=False):
    ops = _ops()
    g = torch.Generator().manual_seed(seed + 7 * B + 11 * Lq + 13 * Lk + H + D)

    def rn(*s):
        return torch.randn(*s, generator=g).to(dev).to(dtype)
    if fused:
        qkv = rn(B, Lq, (H + 2 * Hk) * D)
        q, k, v = (x.unflatten(-1, (-1, D)) for x in qkv.split([H * D, Hk * D, Hk * D], -1))
    else:
        q, k, v = rn(B, Lq, H, D), rn(B, Lk, Hk, D), rn(B, Lk, Hk, D)
    return q, k, v, rn(buckets, H), ops.relpos_bucket_map(buckets, max_distance, bidirectional, dev), rn(B, Lq, H, D)


def check(dev, q, k, v, table, lut, dout, key_mask=None, k_lens=None, causal=False, align_end=False, scale=None, one_bucket=False):
    ops = _ops()
    how = dict(key_mask=key_mask, k_lens=k_lens, causal=causal, align_end=align_end, scale=scale)
    out, lse = ops.relpos_attn_fwd(q, k, v, table, lut, **how)
    dq, dk, dv, dt = ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, **how)
    B, Lq, H, D = q.shape
    Lk = k.shape[1]
    ro, rl, rq, rk, rv = (torch.zeros(x.shape, dtype=F64, device=dev) for x in (q, lse, q, k, v))
    rt = torch.zeros(table.shape, dtype=F64, device=dev)
    for b in range(B):
        n = Lk if k_lens is None else int(k_lens[b])
        seen = torch.arange(Lk, device=dev) < n
        if key_mask is not None:
            seen &= key_mask[b].bool()
        ro[b], rl[b], (rq[b], rk[b], rv[b], t) = ref_attention(q[b], k[b], v[b], table, lut, scale or D ** -0.5, seen,
                                                               (n - Lq if align_end else 0, causal), dout[b])
        rt += t.detach()
    ro, rl = ro.detach(), rl.detach()
    tol = TOL[q.dtype]
    fin = torch.isfinite(rl)
    assert torch.equal(fin, torch.isfinite(lse)) and bool((lse[~fin] == -math.inf).all())
    assert float(((lse.to(F64) - rl)[fin].abs() / rl[fin].abs().clamp(min=1)).max() if fin.any() else 0) < 2e-5
    got = dict(out=rel(out, ro), dq=rel(dq, rq), dk=rel(dk, rk), dv=rel(dv, rv), dtable=rel(dt, rt))
    if one_bucket:
        # every (i, j) in one bucket: sum_j ds_ij = sum_j p dp - delta sum_j p = 0 in exact arithmetic, so there is no value to be relative to.  What is left
        # is the rounding of the summands: tol times their size, sum |ds| <= sum_i 2 max_j |dp_ij| <= 2 rows max |dout| max |v|
        got["dtable"] = float(dt.abs().max()) / (2 * B * Lq * float(dout.float().norm(dim=-1).max()) * float(v.float().norm(dim=-1).max()))
    print(got, flush=True)
    assert max(got.values()) < tol, got
    return out, lse, dq, dk, dv, dt


SHAPES = [  # B, Lq, Lk, H, Hk, D
    (1, 1, 1, 1, 1, 64), (2, 3, 1, 2, 2, 64), (1, 1, 129, 4, 2, 64), (2, 64, 64, 2, 2, 64), (2, 65, 63, 3, 3, 64), (1, 200, 200, 4, 1, 64),
    (2, 127, 385, 2, 1, 32), (1, 300, 300, 2, 2, 8), (1, 90, 130, 2, 2, 40), (1, 130, 257, 4, 2, 128), (2, 70, 70, 2, 2, 96), (3, 513, 513, 8, 8, 64),
    (8, 257, 256, 12, 12, 64), (4, 640, 640, 16, 4, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("causal", [False, True])
def test_forward_and_gradients(dev, shape, dtype, causal):
    """every tile form (16 and 32 columns a wave, head dims padded to 32 / 64 / 128), odd lengths, shared kv heads"""
    print("CASE", shape, dtype, causal, flush=True)
    B, Lq, Lk, H, Hk, D = shape
    q, k, v, table, lut, dout = make(dev, dtype, B, Lq, Lk, H, Hk, D, bidirectional=not causal, fused=Lq == Lk)
    check(dev, q, k, v, table, lut, dout, causal=causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("span", [9, 48, 200, 1024])
def test_bucket_maps(dev, dtype, span):
    """spans below a tile, across tiles, beyond the sequence; both sides used"""
    print("CASE", span, dtype, flush=True)
    q, k, v, table, lut, dout = make(dev, dtype, 2, 450, 450, 2, 2, 64, buckets=16, max_distance=span)
    check(dev, q, k, v, table, lut, dout)
    check(dev, q, k, v, table, lut, dout, causal=True, scale=0.3)


def test_any_map(dev):
    """a map that is no distance scheme at all: one entry (no positions), and an unordered one"""
    ops = _ops()
    q, k, v, table, _, dout = make(dev, torch.float32, 2, 100, 140, 2, 2, 64, buckets=5, max_distance=20)
    check(dev, q, k, v, table, torch.zeros(1, dtype=torch.int32, device=dev) + 3, dout, one_bucket=True)
    lut = torch.randint(0, 5, (41,), generator=torch.Generator().manual_seed(3)).int().to(dev)
    check(dev, q, k, v, table, lut, dout)
    # entries out of range are clamped on the device
    bad = lut.clone(); bad[0], bad[40] = -7, 1 << 20
    good = lut.clone(); good[0], good[40] = 0, 4
    assert torch.equal(ops.relpos_attn_fwd(q, k, v, table, bad)[0], ops.relpos_attn_fwd(q, k, v, table, good)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [False, True])
def test_masks(dev, dtype, causal):
    """holes, a whole masked chunk, an empty sequence, only the last key, and infinities / NaN in every hidden K / V row"""
    print("CASE", dtype, causal, flush=True)
    B, Lk = 6, 333
    q, k, v, table, lut, dout = make(dev, dtype, B, Lk, Lk, 4, 2, 64, seed=5)
    m = torch.ones(B, Lk, dtype=torch.bool)
    m[0] = torch.rand(Lk, generator=torch.Generator().manual_seed(1)) < 0.5
    m[1, 64:200] = False
    m[2] = False
    m[3, :-1] = False
    m[4, 100:] = False
    m = m.to(dev)
    clean = check(dev, q, k, v, table, lut, dout, key_mask=m, causal=causal)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
        kb, vb = k.clone(), v.clone()
        kb[~m], vb[~m] = bad, bad
        ops = _ops()
        out, lse = ops.relpos_attn_fwd(q, kb, vb, table, lut, key_mask=m, causal=causal)
        grads = ops.relpos_attn_bwd(q, kb, vb, table, lut, out, dout, lse, key_mask=m, causal=causal)
        for x, y in zip((out, lse) + grads, clean):
            assert torch.equal(x, y)
    assert not clean[0][2].any() and not clean[2][2].any() and not clean[3][2].any() and not clean[4][2].any()
    # a row-strided uint8 mask says the same
    wide = torch.zeros(B, Lk + 19, dtype=torch.uint8, device=dev)
    wide[:, :Lk] = m.to(torch.uint8) * 3
    assert torch.equal(ops.relpos_attn_fwd(q, k, v, table, lut, key_mask=wide[:, :Lk], causal=causal)[0], clean[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Lq", [1, 5, 16, 17, 40])
def test_cache(dev, dtype, Lq):
    """few queries against caches of unlike fill (none, one key, less than the queries, many): the split form and the plain one; single tokens
    must also agree with the rows of one long causal pass"""
    print("CASE", dtype, Lq, flush=True)
    B, cap = 7, 1500
    q, k, v, table, lut, dout = make(dev, dtype, B, Lq, cap, 8, 2, 128, bidirectional=False, seed=2)
    lens = torch.tensor([0, 1, 3, 513, 1024, 1499, 1500], dtype=torch.int32, device=dev)
    for b in range(B):
        k[b, int(lens[b]):], v[b, int(lens[b]):] = math.nan, math.nan
    for causal in (False, True):
        check(dev, q, k, v, table, lut, dout, k_lens=lens, causal=causal, align_end=True)
    wrong = torch.tensor([-5, 1, 3, 513, 1024, 1499, 1 << 30], dtype=torch.int32, device=dev)         # clamped to [0, cap]
    ops = _ops()
    assert torch.equal(ops.relpos_attn_fwd(q, k, v, table, lut, k_lens=wrong, align_end=True)[0], ops.relpos_attn_fwd(q, k, v, table, lut, k_lens=lens, align_end=True)[0])


def test_single_tokens_follow_a_whole_pass(dev):
    ops = _ops()
    L, H, Hk, D = 700, 4, 2, 64
    q, k, v, table, lut, _ = make(dev, torch.float32, 1, L, L, H, Hk, D, bidirectional=False)
    whole, lse = ops.relpos_attn_fwd(q, k, v, table, lut, causal=True)
    for n in (1, 2, 64, 65, 512, 513, 700):
        one, l1 = ops.relpos_attn_fwd(q[:, n - 1:n], k, v, table, lut, k_lens=torch.tensor([n], dtype=torch.int32, device=dev), causal=True, align_end=True)
        assert rel(one[0, 0], whole[0, n - 1]) < 2e-6 and rel(l1[0, :, 0], lse[0, :, n - 1]) < 2e-6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [False, True])
def test_packed(dev, dtype, causal):
    """ragged sequences (empty ones, one token, across tiles) behind one another equal the sequences alone, bit for bit; rows outside are zero in fresh
    outputs, untouched in given ones; a wrong `longest` changes nothing"""
    print("CASE", dtype, causal, flush=True)
    ops = _ops()
    lens = [0, 1, 5, 64, 0, 131, 300, 2, 0]
    H, Hk, D, tail = 4, 2, 64, 21
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
    T = int(cu[-1]) + tail
    q, k, v, table, lut, dout = (x[0] if x.dim() == 4 else x for x in make(dev, dtype, 1, T, T, H, Hk, D, fused=True, bidirectional=not causal))
    km = (torch.rand(T, generator=torch.Generator().manual_seed(9)) < 0.8).to(dev)
    for mask in (None, km):
        res = []
        for hint in (None, 300, 1, 5000):
            how = dict(cu_q=cu, cu_k=cu, max_q=hint, max_k=hint, causal=causal, key_mask=mask)
            out, lse = ops.relpos_attn_fwd(q, k, v, table, lut, **how)
            res.append((out, lse) + ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, **how))
        for r in res[1:]:
            for i, (x, y) in enumerate(zip(r, res[0])):
                assert torch.equal(x, y) if i != 5 else rel(x, y) < TOL[dtype]        # (dtable: the partials are cut elsewhere)
        out, lse, dq, dk, dv, dt = res[0]
        end = T - tail
        assert not out[end:].any() and not dq[end:].any() and not dk[end:].any() and not dv[end:].any() and bool((lse[:, end:] == -math.inf).all())
        total = torch.zeros(table.shape, dtype=F64, device=dev)
        for b, n in enumerate(lens):
            if not n:
                continue
            s = slice(int(cu[b]), int(cu[b]) + n)
            m = None if mask is None else mask[None, s]
            if m is None or n >= 10:
                a = check(dev, *(x[None, s] for x in (q, k, v)), table, lut, dout[None, s], key_mask=m, causal=causal)
            else:       # (a lone row with one probability near 1 has ds = p1 p2 (dp1 - dp2), small beside the rounding of delta: no bound of 2 u there)
                one = [x[None, s] for x in (q, k, v)]
                a = ops.relpos_attn_fwd(*one, table, lut, key_mask=m, causal=causal)
                a += ops.relpos_attn_bwd(*one, table, lut, a[0], dout[None, s], a[1], key_mask=m, causal=causal)
            for x, y in zip((out[s], lse[:, s], dq[s], dk[s], dv[s]), (a[0][0], a[1][0], a[2][0], a[3][0], a[4][0])):
                assert torch.equal(x, y)
            total += a[5].to(F64)
        assert rel(dt, total) < 2 * TOL[dtype]
    mine = [torch.full_like(x, 7.0) for x in (q, q, k, v)]
    ops.relpos_attn_fwd(q, k, v, table, lut, cu_q=cu, cu_k=cu, out=mine[0], causal=causal)
    ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, cu_q=cu, cu_k=cu, causal=causal, dq=mine[1], dk=mine[2], dv=mine[3])
    for x in mine:
        assert bool((x[end:] == 7.0).all()) and not bool((x[:end] == 7.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1030, 1030, 2, 1, 64), (2, 515, 190, 6, 2, 64), (2, 300, 333, 15, 3, 40), (3, 513, 513, 16, 4, 128), (1, 200, 70, 6, 1, 96)])
@pytest.mark.parametrize("ragged", [False, True])
def test_long_walks_of_shared_heads_in_parts(dev, dtype, shape, ragged):
    """dk and dv of a kv head with many query heads and rows, where few workgroups hold keys: the heads are dealt over several workgroups"""
    print("CASE", dtype, shape, ragged, flush=True)
    B, Lq, Lk, H, Hk, D = shape
    q, k, v, table, lut, dout = make(dev, dtype, *shape)
    lens = torch.tensor([Lk - 61 * (b + 1) if b < 2 else 0 for b in range(B)], dtype=torch.int32, device=dev) if ragged else None
    mask = None
    if ragged:
        mask = torch.rand(B, Lk, generator=torch.Generator().manual_seed(4)).to(dev) < 0.7
        k, v = (torch.where((mask & (torch.arange(Lk, device=dev) < lens[:, None]))[..., None, None], x, math.nan) for x in (k, v))
        want_k = torch.nan_to_num(k)                         # (the oracle sees zeros in hidden rows, the kernels NaN)
        out, lse = _ops().relpos_attn_fwd(q, k, v, table, lut, key_mask=mask, k_lens=lens)
        got = _ops().relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, key_mask=mask, k_lens=lens)
        a = check(dev, q, want_k, torch.nan_to_num(v), table, lut, dout, key_mask=mask, k_lens=lens)
        for x, y in zip((out, lse) + got, a):
            assert torch.equal(x, y)
        return
    a = check(dev, q, k, v, table, lut, dout, causal=Lq == Lk)
    dk = torch.full((B, Hk, Lk, D + 8), 7.0, dtype=dtype, device=dev)[..., :D].permute(0, 2, 1, 3)
    dv = torch.full((B, Lk, Hk, 2, D), 7.0, dtype=dtype, device=dev)
    _ops().relpos_attn_bwd(q, k, v, table, lut, a[0], dout, a[1], causal=Lq == Lk, dq=torch.empty_like(q), dk=dk, dv=dv[:, :, :, 1])
    assert torch.equal(dk, a[3]) and torch.equal(dv[:, :, :, 1], a[4]) and bool((dv[:, :, :, 0] == 7).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(2, 86, 2100, 2, 2, 40), (1, 9, 1300, 8, 4, 64), (3, 128, 1025, 2, 1, 128), (2, 1100, 5, 2, 2, 64), (1, 2500, 128, 4, 2, 64),
                                   (1, 3100, 127, 6, 1, 32), (2, 1025, 64, 2, 2, 96)])
@pytest.mark.parametrize("how", ["plain", "causal", "ragged"])
def test_backward_of_long_against_short(dev, dtype, shape, how):
    """few query rows against many keys, few keys against many query rows: the long side's walk is cut into pieces whose sums are joined"""
    print("CASE", dtype, shape, how, flush=True)
    B, Lq, Lk, H, Hk, D = shape
    q, k, v, table, lut, dout = make(dev, dtype, *shape)
    opt = {}
    if how == "causal":
        opt = dict(causal=True, align_end=Lq < Lk)
    elif how == "ragged":
        opt = dict(k_lens=torch.tensor([max(1, Lk // 3) if b else Lk for b in range(B)], dtype=torch.int32, device=dev),
                   key_mask=torch.rand(B, Lk, generator=torch.Generator().manual_seed(4)).to(dev) < 0.7)
    a = check(dev, q, k, v, table, lut, dout, **opt)
    alone = [x[:1] if torch.is_tensor(x) else x for x in (q, k, v)]
    one = {n: x[:1] if torch.is_tensor(x) else x for n, x in opt.items()}
    got = _ops().relpos_attn_bwd(*alone, table, lut, a[0][:1], dout[:1], a[1][:1].contiguous(), **one)
    if H == Hk:                                             # (the heads of a group are dealt over workgroups by the grid's size)
        for x, y in zip(got[:3], a[2:5]):
            assert torch.equal(x, y[:1])


def test_packed_without_a_sequence(dev):
    """offsets of no sequence at all: fresh outputs are zero, given ones stay as they were"""
    ops = _ops()
    q, k, v, table, lut, dout = (x[0] if x.dim() == 4 else x for x in make(dev, torch.bfloat16, 1, 90, 90, 4, 2, 64))
    cu = torch.zeros(1, dtype=torch.int32, device=dev)
    out, lse = ops.relpos_attn_fwd(q, k, v, table, lut, cu_q=cu, cu_k=cu)
    dq, dk, dv, dt = ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, cu_q=cu, cu_k=cu)
    assert not out.any() and bool((lse == -math.inf).all()) and not dq.any() and not dk.any() and not dv.any() and not dt.any()
    mine = [torch.full_like(x, 7.0) for x in (q, k, v)]
    ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, cu_q=cu, cu_k=cu, dq=mine[0], dk=mine[1], dv=mine[2])
    assert all(bool((x == 7).all()) for x in mine)


def test_options_are_taken_by_value(dev):
    """a scale given as a 0-dim tensor that changes between two calls, gradients into given views where the walk is split"""
    ops = _ops()
    q, k, v, table, lut, dout = make(dev, torch.float32, 1, 70, 2100, 2, 2, 64)
    scale = torch.tensor(0.125)
    one = ops.relpos_attn_fwd(q, k, v, table, lut, scale=scale)[0]
    scale.mul_(2)
    two = ops.relpos_attn_fwd(q, k, v, table, lut, scale=scale)[0]
    assert torch.equal(one, ops.relpos_attn_fwd(q, k, v, table, lut, scale=0.125)[0])
    assert torch.equal(two, ops.relpos_attn_fwd(q, k, v, table, lut, scale=0.25)[0]) and not torch.equal(one, two)
    from spokennlp_amd import relpos
    grads = []
    for s in (scale, 0.25):                                 # (the tensor changes between the forward pass and the backward one)
        leaf = q.detach().clone().requires_grad_()
        y = relpos.relpos_attention(leaf, k, v, table, lut, scale=s)
        scale.fill_(0.5)
        y.backward(dout)
        grads.append(leaf.grad)
    assert torch.equal(*grads)
    out, lse = ops.relpos_attn_fwd(q, k, v, table, lut)
    want = ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse)
    dq = torch.full((1, 2, 70, 72), 7.0, device=dev)[..., :64].permute(0, 2, 1, 3)
    got = ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, dq=dq, dk=torch.empty_like(k), dv=torch.empty_like(v))
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_packed_rows_in_front(dev):
    """offsets that do not start at 0: the rows in front belong to no sequence either"""
    ops = _ops()
    q, k, v, table, lut, dout = (x[0] if x.dim() == 4 else x for x in make(dev, torch.float32, 1, 90, 90, 4, 2, 64))
    cu, at0 = torch.tensor([17, 60, 80], dtype=torch.int32, device=dev), torch.tensor([0, 43, 63], dtype=torch.int32, device=dev)
    out, lse = ops.relpos_attn_fwd(q, k, v, table, lut, cu_q=cu, cu_k=cu)
    grads = ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, cu_q=cu, cu_k=cu)
    o2, l2 = ops.relpos_attn_fwd(q[17:80], k[17:80], v[17:80], table, lut, cu_q=at0, cu_k=at0)
    g2 = ops.relpos_attn_bwd(q[17:80], k[17:80], v[17:80], table, lut, o2, dout[17:80], l2, cu_q=at0, cu_k=at0)
    for x, y in zip((out,) + grads[:3], (o2,) + g2[:3]):
        assert torch.equal(x[17:80], y) and not x[:17].any() and not x[80:].any()
    assert torch.equal(lse[:, 17:80], l2) and bool((lse[:, :17] == -math.inf).all()) and rel(grads[3], g2[3]) < 2e-5


def test_offsets_past_32_bits(dev):
    """a cache whose sequences start more than 2^31 elements apart, keys broadcast over heads by a stride of 0"""
    ops = _ops()
    cap, Hk, D = 1 << 24, 2, 64                              # 2^31 elements a sequence
    big = torch.empty(2 * cap * Hk * D, dtype=torch.bfloat16, device=dev)
    kv = big.view(2, cap, Hk, D)
    q, k, v, table, lut, dout = make(dev, torch.bfloat16, 2, 3, 700, 4, 2, 64)
    kv[:, cap - 700:] = k
    far = kv[:, cap - 700:]
    assert far.stride(0) == 1 << 31
    out, lse = ops.relpos_attn_fwd(q, far, v, table, lut)
    want, wl = ops.relpos_attn_fwd(q, k, v, table, lut)
    assert torch.equal(out, want) and torch.equal(lse, wl)
    q2 = torch.randn(2, 200, 4, D, device=dev).bfloat16()
    out, lse = ops.relpos_attn_fwd(q2, far, v, table, lut)
    want, wl = ops.relpos_attn_fwd(q2, k, v, table, lut)
    assert torch.equal(out, want)
    for x, y in zip(ops.relpos_attn_bwd(q2, far, v, table, lut, out, q2, lse), ops.relpos_attn_bwd(q2, k, v, table, lut, want, q2, wl)):
        assert torch.equal(x, y)
    del big, kv, far
    one = k[:, :, :1]
    a = ops.relpos_attn_fwd(q2, one.expand(-1, -1, 2, -1), v, table, lut)[0]
    assert torch.equal(a, ops.relpos_attn_fwd(q2, one.expand(-1, -1, 2, -1).contiguous(), v, table, lut)[0])


def test_infinite_table_entries_hide_a_bucket(dev):
    """a bucket at -inf: its keys have p = 0 in forward and backward, near and far, and no gradient; a row whose every key is in it is empty"""
    ops = _ops()
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v, table, lut, dout = make(dev, dtype, 2, 300, 400, 2, 2, 64, buckets=8, max_distance=48)
        table = table.clone()
        table[3], table[7, 1] = -math.inf, -math.inf         # far left for both heads, far right for the second
        finite = torch.isfinite(table)
        out, lse = ops.relpos_attn_fwd(q, k, v, table, lut)
        g = ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse)
        r = torch.arange(400, device=dev)[None] - torch.arange(300, device=dev)[:, None]
        b = table.to(F64)[lut.long()[r.clamp(-48, 48) + 48]].permute(2, 0, 1)
        qq, kk, vv = (x.to(F64).requires_grad_(True) for x in (q, k, v))
        p = torch.softmax(torch.einsum("bihd,bjhd->bhij", qq, kk) / 8 + b, -1)
        o = torch.einsum("bhij,bjhd->bihd", p, vv)
        o.backward(dout.to(F64))
        assert max(rel(x, y) for x, y in zip((out,) + g[:3], (o.detach(), qq.grad, kk.grad, vv.grad))) < TOL[dtype]
        assert not g[3][~finite].any() and bool(torch.isfinite(g[3]).all())
        table[:] = -math.inf
        out, lse = ops.relpos_attn_fwd(q, k, v, table, lut)
        g = ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse)
        assert not any(x.any() for x in (out,) + g) and bool((lse == -math.inf).all())


def test_packed_with_bad_offsets_stays_inside(dev):
    """offsets that run backwards or past the buffers are clamped on the device: some rows are wrong, none outside is touched"""
    ops = _ops()
    T = 200
    q, k, v, table, lut, dout = (x[0] if x.dim() == 4 else x for x in make(dev, torch.bfloat16, 1, T, T, 2, 2, 64))
    guard = torch.full((3 * T, 2, 64), 7.0, dtype=torch.bfloat16, device=dev)
    cu = torch.tensor([-50, 90, 40, 1 << 30], dtype=torch.int32, device=dev)
    out, lse = ops.relpos_attn_fwd(q, k, v, table, lut, cu_q=cu, cu_k=cu, out=guard[T:2 * T])
    ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, cu_q=cu, cu_k=cu, dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    assert bool((guard[:T] == 7).all()) and bool((guard[2 * T:] == 7).all()) and bool(torch.isfinite(guard).all())


def test_gradients_against_differences(dev):
    """a directional derivative of sum(out * w) from the kernels' own forward, fp32: central difference, step 2^-7 along a unit-ish direction; the error of
    the quotient is third order in the step plus 2^-24 / step relative to the sum: 2e-3 relative covers both"""
    ops = _ops()
    q, k, v, table, lut, w = make(dev, torch.float32, 2, 90, 110, 4, 2, 32)
    out, lse = ops.relpos_attn_fwd(q, k, v, table, lut)
    grads = ops.relpos_attn_bwd(q, k, v, table, lut, out, w, lse)
    xs = [q, k, v, table]
    for n in range(4):
        g = torch.Generator().manual_seed(n)
        d = torch.randn(xs[n].shape, generator=g).to(dev)
        h = 2.0 ** -7
        f = []
        for sgn in (1, -1):
            y = list(xs)
            y[n] = xs[n] + sgn * h * d
            f.append((ops.relpos_attn_fwd(*y, lut)[0].to(F64) * w.to(F64)).sum())
        num, ana = float((f[0] - f[1]) / (2 * h)), float((grads[n].to(F64) * d.to(F64)).sum())
        scale = float(grads[n].norm() * d.norm()) / math.sqrt(d.numel()) + abs(num)
        assert abs(num - ana) < 2e-3 * scale, (n, num, ana)


def test_strided_inputs_and_outputs(dev):
    """a cache laid out [B, heads, capacity, D], gradients written into column blocks of one buffer, a table of another type than the activations"""
    ops = _ops()
    B, L, H, D = 2, 150, 4, 64
    q, k, v, table, lut, dout = make(dev, torch.bfloat16, B, L, L, H, H, D, fused=True)
    out, lse = ops.relpos_attn_fwd(q, k, v, table, lut)
    base = ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse)
    kt, vt = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
    assert torch.equal(ops.relpos_attn_fwd(q, kt, vt, table, lut)[0], out)
    dqkv = torch.full((B, L, 3 * H * D), 9.0, dtype=torch.bfloat16, device=dev)
    blocks = [x.unflatten(-1, (H, D)) for x in dqkv.split(H * D, -1)]
    got = ops.relpos_attn_bwd(q, kt, vt, table, lut, out, dout.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), lse, dq=blocks[0], dk=blocks[1], dv=blocks[2])
    for x, y in zip(blocks, base):
        assert torch.equal(x, y)
    assert torch.equal(got[3], base[3])
    assert torch.equal(ops.relpos_attn_fwd(q, k, v, table.float(), lut)[0], out)
    t32 = ops.relpos_attn_bwd(q, k, v, table.float(), lut, out, dout, lse)[3]
    assert t32.dtype == torch.float32 and torch.equal(t32.bfloat16(), base[3])
    assert ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, need_dtable=False)[3] is None


def test_same_bits_every_time_and_in_any_batch(dev):
    ops = _ops()
    q, k, v, table, lut, dout = make(dev, torch.bfloat16, 8, 400, 400, 12, 12, 64)
    out, lse = ops.relpos_attn_fwd(q, k, v, table, lut)
    a = ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse)
    for _ in range(3):
        b = ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    o1, l1 = ops.relpos_attn_fwd(q[3:4], k[3:4], v[3:4], table, lut)
    b = ops.relpos_attn_bwd(q[3:4], k[3:4], v[3:4], table, lut, o1, dout[3:4], l1)
    assert torch.equal(o1[0], out[3]) and torch.equal(l1[0], lse[3]) and all(torch.equal(x[0], y[3]) for x, y in zip(b[:3], a[:3]))


def test_graph_replay_and_streams(dev):
    """captured and replayed (twice the same graph pool, two graphs alive at once, eager work between), and on a side stream"""
    ops = _ops()
    sets = []
    for n, (B, L, D) in enumerate(((2, 200, 64), (1, 700, 64), (2, 300, 128))):        # (D = 128: more than 64 KiB of LDS, asked for at every launch)
        q, k, v, table, lut, dout = make(dev, torch.bfloat16, B, L, L, 4, 2, D, seed=n)
        tok = torch.randn(B, 1, 4, D, device=dev).bfloat16()

        def step(q=q, k=k, v=v, table=table, lut=lut, dout=dout, tok=tok):
            out, lse = ops.relpos_attn_fwd(q, k, v, table, lut, causal=True)
            one, _ = ops.relpos_attn_fwd(tok, k, v, table, lut, align_end=True)
            return (out, lse, one) + ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, causal=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        sets.append((q, step, graph, got, want))
    for i in range(4):
        for q, step, graph, got, want in sets:
            if i == 2:
                q.mul_(0.5)
            want = step()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want)), i


@pytest.mark.parametrize("B,H,Lq,Lk,span", [(1, 1, 1, 1, 128), (2, 3, 5, 7, 9), (3, 2, 64, 512, 48), (2, 12, 333, 257, 128), (1, 2, 700, 1201, 200), (4, 1, 130, 9, 1024)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dense_bias_and_gradient(dev, B, H, Lq, Lk, span, dtype):
    ops = _ops()
    print("CASE", B, H, Lq, Lk, span, dtype, flush=True)
    g = torch.Generator().manual_seed(B + Lq)
    table = torch.randn(32, H, generator=g).to(dev)
    lut = ops.relpos_bucket_map(32, span, True, dev)
    for off in (0, 40, -13):
        r = torch.arange(Lk, device=dev)[None] - torch.arange(Lq, device=dev)[:, None] - off
        bucket = lut.long()[r.clamp(-span, span) + span]
        assert torch.equal(ops.relpos_bias_fwd(table, lut, Lq, Lk, q_offset=off, out_dtype=dtype), table[bucket].permute(2, 0, 1).to(dtype))
        d = torch.randn(B, H, Lq, Lk, generator=g).to(dev).to(dtype)
        want = torch.zeros(H, 32, dtype=F64, device=dev).index_add_(1, bucket.flatten(), d.to(F64).sum(0).flatten(1)).t()
        mass = torch.zeros(H, 32, dtype=F64, device=dev).index_add_(1, bucket.flatten(), d.to(F64).abs().sum(0).flatten(1)).t()
        got = ops.relpos_bias_bwd(d, lut, 32, q_offset=off)
        assert bool(((got.to(F64) - want).abs() <= 2e-6 * mass).all())              # a tree of fp32 sums: some tens of 2^-24 times the summed sizes
        assert torch.equal(got, ops.relpos_bias_bwd(d, lut, 32, q_offset=off))
        if B == 1:
            assert torch.equal(got, ops.relpos_bias_bwd(d[0], lut, 32, q_offset=off))
    # masked scores arrive as exact zeros next to infinities elsewhere in other heads: a head's sum is its own
    if H > 1 and Lq > 1:
        d = torch.ones(B, H, Lq, Lk, device=dev, dtype=dtype)
        d[:, 0] = math.inf
        got = ops.relpos_bias_bwd(d, lut, 32)
        assert bool(torch.isfinite(got[:, 1:]).all())


def test_empty_calls(dev):
    ops = _ops()
    lut = ops.relpos_bucket_map(32, 128, True, dev)
    table = torch.randn(32, 4, device=dev)
    for Bq, Lq, Lk in ((0, 5, 5), (2, 0, 5), (2, 5, 0), (0, 0, 0)):
        q, k = torch.randn(Bq, Lq, 4, 64, device=dev), torch.randn(Bq, Lk, 4, 64, device=dev)
        out, lse = ops.relpos_attn_fwd(q, k, k, table, lut)
        dq, dk, dv, dt = ops.relpos_attn_bwd(q, k, k, table, lut, out, torch.ones_like(q), lse)
        for x in (out, dq, dk, dv, dt):
            assert not x.any()
        assert bool((lse == -math.inf).all())
        assert not ops.relpos_bias_bwd(torch.zeros(Bq, 4, Lq, Lk, device=dev), lut, 32).any()
        assert ops.relpos_bias_fwd(table, lut, Lq, Lk).shape == (4, Lq, Lk)
    cu = torch.zeros(1, dtype=torch.int32, device=dev)
    q = torch.randn(5, 4, 64, device=dev)
    out, lse = ops.relpos_attn_fwd(q, q, q, table, lut, cu_q=cu, cu_k=cu)
    assert not out.any() and not any(x.any() for x in ops.relpos_attn_bwd(q, q, q, table, lut, out, q, lse, cu_q=cu, cu_k=cu))


# ------------------------------------------------------------------------------------------------ differentiable surface
def test_autograd_functions(dev):
    """gradients through torch autograd: q / k / v leaves, a fused projection (padded, packed with rows outside), the dense bias; dout of any strides"""
    from spokennlp_amd import relpos as R
    ops = _ops()
    q, k, v, table, lut, dout = make(dev, torch.float32, 2, 70, 90, 4, 2, 64)
    out, lse = ops.relpos_attn_fwd(q, k, v, table, lut)
    want = ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, table)]
    R.relpos_attention(*leaves, lut).backward(dout.transpose(1, 3).contiguous().transpose(1, 3))      # last dimension strided
    assert all(torch.equal(x.grad, y) for x, y in zip(leaves, want))
    # an expanded dout (the gradient of a sum)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, table)]
    R.relpos_attention(*leaves, lut).sum().backward()
    ones = ops.relpos_attn_bwd(q, k, v, table, lut, out, torch.ones_like(out), lse)
    assert all(torch.equal(x.grad, y) for x, y in zip(leaves, ones))
    # only some leaves
    t = table.clone().requires_grad_(True)
    R.relpos_attention(q, k, v, t, lut).backward(dout)
    assert torch.equal(t.grad, want[3])
    with torch.no_grad():
        assert torch.equal(R.relpos_attention(q, k, v, table, lut), out)
    # fused, packed
    lens, H, Hk, D = [33, 0, 70], 4, 2, 64
    cu = torch.tensor([0, 33, 33, 103], dtype=torch.int32, device=dev)
    qkv = torch.randn(110, (H + 2 * Hk) * D, generator=torch.Generator().manual_seed(1)).to(dev)
    d = torch.randn(110, H * D, generator=torch.Generator().manual_seed(2)).to(dev)
    a, t = qkv.clone().requires_grad_(True), table.clone().requires_grad_(True)
    y = R.relpos_self_attention(a, H, t, lut, kv_heads=Hk, cu_seqlens=cu, longest=70)
    y.backward(d)
    assert not y[103:].any() and not a.grad[103:].any() and bool(torch.isfinite(a.grad).all())
    b, t2 = qkv.clone().requires_grad_(True), table.clone().requires_grad_(True)
    parts = [R.relpos_self_attention(b[None, s:e], H, t2, lut, kv_heads=Hk) for s, e in ((0, 33), (33, 103))]
    torch.cat([p[0] for p in parts]).backward(d[:103])
    assert torch.equal(a.grad[:103], b.grad[:103]) and rel(t.grad, t2.grad) < 2e-5
    # dense bias feeding composed attention equals the fused one
    t3 = table.clone().requires_grad_(True)
    s = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(2, 2)) * 64 ** -0.5 + R.relpos_bias(t3, lut, 70, 90)
    o = torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), v.repeat_interleave(2, 2))
    o.backward(dout)
    assert rel(o, out) < 2e-5 and rel(t3.grad, want[3]) < 2e-5


def test_layers_together_and_a_training_step(dev):
    """two layers that share one table, bf16 module under the framework's own optimiser kernel: forward and every gradient against the same layers composed
    in 64 bits; padded and packed inputs give the same tokens"""
    from spokennlp_amd import relpos as R
    ops = _ops()
    torch.manual_seed(0)
    Hs, heads, L, lens = 256, 4, 150, [150, 97, 1]
    l0 = R.RelPosSelfAttention(Hs, heads, kv_heads=2).to(dev)
    l1 = R.RelPosSelfAttention(Hs, heads, kv_heads=2, table=l0.table).to(dev)
    assert l1.table is l0.table and len(list(torch.nn.ModuleList([l0, l1]).parameters())) == 9
    x = torch.randn(3, L, Hs, device=dev)
    mask = torch.arange(L, device=dev)[None] < torch.tensor(lens, device=dev)[:, None]
    w = torch.randn(3, L, Hs, device=dev) * mask[..., None]

    def run(xx, **kw):
        h = xx + l0(xx, **kw)
        return h + l1(h, **kw)
    y = run(x, key_mask=mask)
    (y * w).sum().backward()
    grads = {n: p.grad.clone() for n, p in torch.nn.ModuleList([l0, l1]).named_parameters()}
    # packed
    cu = torch.tensor([0, 150, 247, 248], dtype=torch.int32, device=dev)
    yp = run(x[mask], cu_seqlens=cu, longest=150)
    assert rel(yp, y[mask]) < 2e-6
    # 64 bits
    P = {n: p.detach().to(F64).requires_grad_(True) for n, p in torch.nn.ModuleList([l0, l1]).named_parameters()}

    def layer(h, i):
        qkv = h @ P[f"{i}.qkv.weight"].t() + P[f"{i}.qkv.bias"]
        q, k, v = (t.unflatten(-1, (-1, 64)) for t in qkv.split([256, 128, 128], -1))
        r = torch.arange(L, device=dev)[None] - torch.arange(L, device=dev)[:, None]
        b = P["0.table"][l0.bucket_map.long()[r.clamp(-128, 128) + 128]].permute(2, 0, 1)
        s = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(2, 2)) / 8 + b
        p = torch.softmax(s.masked_fill(~mask[:, None, None], -math.inf), -1)
        return torch.einsum("bhij,bjhd->bihd", p, v.repeat_interleave(2, 2)).flatten(-2) @ P[f"{i}.out.weight"].t() + P[f"{i}.out.bias"]
    h = x.to(F64)
    h = h + layer(h, 0)
    h = h + layer(h, 1)
    assert rel(y * mask[..., None], h.detach() * mask[..., None]) < 2e-5
    (h * w.to(F64)).sum().backward()
    for n, g in grads.items():
        assert rel(g, P[n].grad) < 5e-5, n                   # two layers of fp32 products, each within 2e-5
    # one optimiser step of the shared table and its gradient through amdseg_adamw
    p, m, v2 = l0.table.detach().clone().flatten(), torch.zeros(128, device=dev), torch.zeros(128, device=dev)
    ops.adamw(p, grads["0.table"].flatten().contiguous(), m, v2, None, 1e-2, 0.9, 0.999, 1e-8, 0.0, 1)
    assert bool(((p - l0.table.detach().flatten()).abs() <= 1.0001e-2).all()) and bool((p != l0.table.detach().flatten()).any())


def test_backward_captured_beside_a_living_eager_graph(dev):
    """a training step captured into a graph while an eager graph of the same leaves is alive (its buffers held): both finish, with the same gradients"""
    from spokennlp_amd import relpos as R
    q, k, v, table, lut, dout = make(dev, torch.bfloat16, 2, 130, 130, 4, 2, 64)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, table)]
    eager = R.relpos_attention(*leaves, lut)
    copies = [x.detach().clone().requires_grad_(True) for x in leaves]

    def step():
        o = R.relpos_attention(*copies, lut)
        return torch.autograd.grad(o, copies, dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    eager.backward(dout)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y.grad) for x, y in zip(got, leaves))
