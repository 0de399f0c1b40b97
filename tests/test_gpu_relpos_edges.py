"""Attention under a learned relative position bias where calls are at the edge of what the documentation allows, on a real MI355X.  The oracle and the
tolerances are those of test_gpu_relpos.py unless a test says otherwise."""
import math

import pytest
import torch

from tests.test_gpu_relpos import F64, TOL, _ops, check, make, rel

pytestmark = pytest.mark.gpu


def passes(q, k, v, table, lut, dout, **how):
    """forward and backward: out, lse, dq, dk, dv, dtable"""
    ops = _ops()
    out, lse = ops.relpos_attn_fwd(q, k, v, table, lut, **how)
    return (out, lse) + ops.relpos_attn_bwd(q, k, v, table, lut, out, dout, lse, **how)


# ---- finite table entries of any size
# What |s| ~ 2^15 costs: the entry over the scale, the sums of the products on top of it, lse and its product with log2 e are rounded to 24 bits there, half a step
# of [2^14, 2^15) is 2^-10, at most eight of them (four products of 32 at D <= 128, or one addition in fp32, and four others) reach the exponent: e^(8 * 2^-10) - 1
FAR_TOL = 8 * 2.0 ** -10


def one_key(out, v):
    """a row with all of its probability on one key: e v / e with e near 1 rounded where it is summed, 1 / e and two products: four roundings of the row's v in fp32;
    in bf16 e is rounded too, but the sum 1 / e is taken of is not: one of 2^-8 more (and the output's own)"""
    tol = 4 * 2.0 ** -24 if out.dtype == torch.float32 else 2 * 2.0 ** -8
    return bool(((out.to(F64) - v.to(F64)).abs() <= tol * v.to(F64).abs()).all())


def ref_shifted(q, k, v, table, lut, seen, causal, dout):
    """ref_attention with each row's largest visible entry taken off first: the same softmax, and 64 bits then hold the products beside entries of any size"""
    span = lut.numel() // 2
    q, k, v, table = (x.detach().to(F64).requires_grad_() for x in (q, k, v, table))
    r = torch.arange(k.shape[0], device=q.device)[None] - torch.arange(q.shape[0], device=q.device)[:, None]
    b = table[lut.long()[r.clamp(-span, span) + span]].permute(2, 0, 1)
    vis = seen[None] & (r <= 0) if causal else seen[None].expand_as(r)
    top = b.detach().masked_fill(~vis[None], -math.inf).amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    s = torch.einsum("ihd,jhd->hij", q, k) * q.shape[-1] ** -0.5 + (b - top)
    blind = ~vis.any(1)
    p = torch.softmax(s.masked_fill(~vis[None], -math.inf).masked_fill(blind[None, :, None], 0.0), -1) * (~blind)[None, :, None]
    out = torch.einsum("hij,jhd->ihd", p, v)
    return [out.detach()] + list(torch.autograd.grad(out, (q, k, v, table), dout.to(F64)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("entry", ["lowest", "lowest_bf16", -1e30, -1e9, -1e4, 1e4, 1e9, "highest_bf16", "highest"])
@pytest.mark.parametrize("where", ["near", "far"])
def test_finite_table_entries_of_any_size(dev, dtype, entry, where):
    """a bucket at the types' lowest (highest) value: it loses against (wins over) every other one, and a row that sees nothing else has the softmax over it, with
    its gradients.  near: the bucket of distance 0, under a causal mask (row 0 sees nothing else); far: the last bucket to the left, most rows see
    nothing else"""
    print("CASE", dtype, entry, where, flush=True)
    x = {"lowest": torch.finfo(torch.float32).min, "lowest_bf16": torch.finfo(torch.bfloat16).min, "highest": torch.finfo(torch.float32).max,
         "highest_bf16": torch.finfo(torch.bfloat16).max}.get(entry, entry)
    causal = where == "near"
    q, k, v, table, lut, dout = make(dev, dtype, 1, 200, 200, 2, 2, 64, buckets=8, max_distance=48, bidirectional=not causal)
    table = table.float()
    seen = torch.ones(200, dtype=torch.bool, device=dev)
    if causal:
        table[0] = x
        if x > 0:
            table[3] = x                                     # (two buckets that win: both are seen by most rows)
    else:
        table[int(lut[0])] = x
        seen[30:] = False
    got = passes(q, k, v, table, lut, dout, causal=causal, key_mask=seen[None])
    assert all(bool(torch.isfinite(y).all()) for y in got)
    want = ref_shifted(q[0], k[0], v[0], table, lut, seen, causal, dout[0])
    err = dict(out=rel(got[0][0], want[0]), dq=rel(got[2][0], want[1]), dk=rel(got[3][0], want[2]), dv=rel(got[4][0], want[3]))
    # dtable: a row whose probability is all in one bucket gives it sum_j ds_ij = 0 in exact arithmetic; relative to the summands' size (test_any_map)
    mass = 2 * 200 * float(dout.float().norm(dim=-1).max()) * float(v.float().norm(dim=-1).max())
    err["dtable"] = float((got[5].to(F64) - want[4]).abs().max()) / mass
    print(err, flush=True)
    assert max(err.values()) < TOL[dtype] + FAR_TOL, err
    if causal and x < 0:
        assert one_key(got[0][0, 0], v[0, 0])
    # a module's dense bias has the entry itself
    assert torch.equal(_ops().relpos_bias_fwd(table, lut, 3, 3)[0, 2, 2], table[int(lut[48]), 0])


def test_finite_table_entries_keep_their_order(dev):
    """of buckets at unlike huge values the largest takes the row"""
    q, k, v, _, _, _ = make(dev, torch.float32, 1, 40, 40, 1, 1, 64)
    lut = torch.tensor([0] * 39 + [1] + [2] * 39, dtype=torch.int32, device=dev)          # left, itself, right
    levels = [torch.finfo(torch.float32).min, -1e38, -4e37, -1e30, -1e9, -2e5, -1e5, -1e4, 0.0, 1e4, 3e4, 1e9, 1e30, 4e37, 1e38, torch.finfo(torch.float32).max]
    for lo, hi in zip(levels, levels[1:]):
        table = torch.tensor([[lo], [hi], [lo]], dtype=torch.float32, device=dev)
        out, lse = _ops().relpos_attn_fwd(q, k, v, table, lut)
        assert one_key(out, v), (lo, hi)
        assert bool(torch.isfinite(lse).all())


# ---- keys that no row sees
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(2, 100, 333, 4, 2, 64), (1, 1, 700, 8, 2, 128), (2, 3, 2100, 4, 2, 64), (2, 90, 2100, 2, 2, 40), (1, 300, 420, 2, 2, 128),
                                   (1, 128, 129, 12, 12, 64), (1, 1, 2, 1, 1, 8)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_keys_behind_the_last_query_are_not_used(dev, dtype, shape, bad):
    """a causal pass over the first Lq places of longer K / V buffers whose rest was never written: the same bits as with finite rows there, their gradients zero"""
    print("CASE", dtype, shape, bad, flush=True)
    B, Lq, Lk, H, Hk, D = shape
    q, k, v, table, lut, dout = make(dev, dtype, *shape, bidirectional=False)
    clean = check(dev, q, k, v, table, lut, dout, causal=True) if Lq > 1 else passes(q, k, v, table, lut, dout, causal=True)
    kb, vb = k.clone(), v.clone()
    kb[:, Lq:], vb[:, Lq:] = bad, bad
    for x, y in zip(passes(q, kb, vb, table, lut, dout, causal=True), clean):
        assert torch.equal(x, y)
    assert not clean[3][:, Lq:].any() and not clean[4][:, Lq:].any()
    # the same with a key mask, and packed with more keys than queries
    m = torch.rand(B, Lk, generator=torch.Generator().manual_seed(3)).to(dev) < 0.8
    m[:, 0] = True
    a, b = passes(q, k, v, table, lut, dout, causal=True, key_mask=m), passes(q, kb, vb, table, lut, dout, causal=True, key_mask=m)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    cq = torch.arange(B + 1, dtype=torch.int32, device=dev) * Lq
    ck = torch.arange(B + 1, dtype=torch.int32, device=dev) * Lk
    flat = [x.flatten(0, 1) for x in (q, k, v, dout)], [x.flatten(0, 1) for x in (q, kb, vb, dout)]
    a, b = (passes(*x[:3], table, lut, x[3], causal=True, cu_q=cq, cu_k=ck) for x in flat)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 300, 310, 2, 2, 64), (1, 640, 670, 48, 48, 64), (2, 300, 399, 4, 2, 128)])
def test_rows_of_a_block_take_nothing_from_keys_behind_it(dev, dtype, shape):
    """causal with the last query at the last key: NaN in keys behind what a block of 128 rows sees leaves those rows as they were"""
    print("CASE", dtype, shape, flush=True)
    B, Lq, Lk, H, Hk, D = shape
    q, k, v, table, lut, dout = make(dev, dtype, *shape, bidirectional=False)
    a = passes(q, k, v, table, lut, dout, causal=True, align_end=True)
    kb, vb = k.clone(), v.clone()
    kb[:, 128 + Lk - Lq:], vb[:, 128 + Lk - Lq:] = math.nan, math.nan
    b = passes(q, kb, vb, table, lut, dout, causal=True, align_end=True)
    for x, y in zip((a[0][:, :128], a[1][:, :, :128], a[2][:, :128]), (b[0][:, :128], b[1][:, :, :128], b[2][:, :128])):
        assert torch.equal(x, y)


# ---- rows that see no key
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(3, 300, 300, 4, 2, 64), (2, 200, 90, 2, 2, 128), (2, 1500, 100, 4, 2, 64), (3, 40, 2100, 4, 4, 32), (3, 9, 700, 2, 2, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_the_gradient_of_a_row_without_a_key_is_not_used(dev, dtype, shape, bad):
    """causal with the first keys hidden, and more queries than keys ending together: rows without a key have q and dout of any value and give no gradient"""
    print("CASE", dtype, shape, bad, flush=True)
    B, Lq, Lk, H, Hk, D = shape
    q, k, v, table, lut, dout = make(dev, dtype, *shape, bidirectional=False)
    m = torch.ones(B, Lk, dtype=torch.bool, device=dev)
    first = [0, 37, 70, 5][:B] if Lk > 90 else [0, 21]
    for b, n in enumerate(first):
        m[b, :n] = False
    if B == 3:
        m[2] = False                                         # (a sequence of no keys at all)
    how = dict(causal=True, align_end=True, key_mask=m)
    a = passes(q, k, v, table, lut, dout, **how)
    empty = (a[1] == -math.inf).all(1)                       # [B, Lq]
    assert empty.any() and not empty.all()
    qb, db = q.clone(), dout.clone()
    qb[empty], db[empty] = bad, bad
    b = passes(qb, k, v, table, lut, db, **how)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    assert not b[2][empty].any()
    cq, ck = (torch.arange(B + 1, dtype=torch.int32, device=dev) * n for n in (Lq, Lk))
    how = dict(causal=True, align_end=True, key_mask=m.flatten(), cu_q=cq, cu_k=ck)
    a, b = (passes(x.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), table, lut, y.flatten(0, 1), **how) for x, y in ((q, dout), (qb, db)))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---- the same bits in any batch
@pytest.mark.parametrize("span", [9, 48, 128, 200])
@pytest.mark.parametrize("extra", [0, 10, 33])
@pytest.mark.parametrize("D", [64, 40, 96])
def test_bits_do_not_follow_the_batch(dev, span, extra, D):
    """a sequence alone (16 query rows a wave) and among 24 (32 rows a wave), whole and packed with hints of any size; spans and offsets that are no multiple of
    a tile"""
    print("CASE", span, extra, D, flush=True)
    L = 400
    q, k, v, table, lut, dout = make(dev, torch.bfloat16, 24, L, L + extra, 12, 12, D, buckets=8, max_distance=span)
    for causal in (False, True):
        how = dict(causal=causal, align_end=True)
        a = passes(q, k, v, table, lut, dout, **how)
        for b in (0, 5):
            one = passes(q[b:b + 1], k[b:b + 1], v[b:b + 1], table, lut, dout[b:b + 1], **how)
            for n in range(5):
                assert torch.equal(one[n][0], a[n][b]), (causal, n)
    cq, ck = (torch.arange(25, dtype=torch.int32, device=dev) * n for n in (L, L + extra))
    flat = [x.flatten(0, 1) for x in (q, k, v)]
    for hint in (None, L + extra, 1):
        p = passes(*flat, table, lut, dout.flatten(0, 1), cu_q=cq, cu_k=ck, max_q=hint, max_k=hint, **how)
        assert torch.equal(p[0], a[0].flatten(0, 1)) and torch.equal(p[1], a[1].transpose(0, 1).flatten(1)), hint
        for n in (2, 3, 4):
            assert torch.equal(p[n], a[n].flatten(0, 1)), (hint, n)


def test_bits_of_single_tokens_in_a_batch_of_any_size(dev):
    """single tokens of more (sequence, kv head) pairs than a grid's second dimension holds"""
    B, H, Hk, D = 16400, 8, 4, 16
    q, k, v, table, lut, _ = make(dev, torch.bfloat16, B, 1, 70, H, Hk, D, buckets=8, max_distance=48)
    out, lse = _ops().relpos_attn_fwd(q, k, v, table, lut, align_end=True)
    for s in (slice(0, 50), slice(8000, 8060), slice(B - 50, B)):
        o, l = _ops().relpos_attn_fwd(q[s], k[s], v[s], table, lut, align_end=True)
        assert torch.equal(o, out[s]) and torch.equal(l, lse[s])


# ---- gradients that torch hands on
def test_gradients_that_start_anywhere(dev):
    """dout as a slice of a larger contiguous gradient: contiguous, and on no 16 bytes"""
    from spokennlp_amd import relpos as R
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, table, lut, dout = make(dev, dtype, 2, 70, 70, 4, 2, 64, fused=True)
        want = passes(q, k, v, table, lut, dout)
        for pad in (1, 3, 7):
            leaves = [x.clone().requires_grad_(True) for x in (q, k, v, table)]
            y = torch.cat([torch.zeros(pad, dtype=dtype, device=dev), R.relpos_attention(*leaves, lut).flatten()])
            y.backward(torch.cat([torch.ones(pad, dtype=dtype, device=dev), dout.flatten()]))
            for x, g in zip(leaves, want[2:]):
                assert torch.equal(x.grad, g)
            qkv = torch.cat([x.flatten(-2) for x in (q, k, v)], -1).requires_grad_(True)
            y = torch.cat([torch.zeros(pad, dtype=dtype, device=dev), R.relpos_self_attention(qkv, 4, table, lut, kv_heads=2).flatten()])
            y.backward(torch.cat([torch.ones(pad, dtype=dtype, device=dev), dout.flatten()]))
            assert torch.equal(qkv.grad, torch.cat([x.flatten(-2) for x in want[2:5]], -1))


# ---- packed batches without a hint, and with one long sequence among short ones
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [False, True])
def test_packed_hints_change_nothing_at_all(dev, dtype, causal):
    """many short sequences and one long one (and empty ones, rows in front and behind): every hint gives the same bits, dtable's too, and the padded call's rows"""
    print("CASE", dtype, causal, flush=True)
    g = torch.Generator().manual_seed(7)
    lens = torch.randint(0, 40, (300,), generator=g).tolist()
    lens[41], lens[42], lens[299] = 1300, 0, 129
    cu = [11]
    for n in lens:
        cu.append(cu[-1] + n)
    H, Hk, D, T = 4, 2, 64, cu[-1] + 50
    cut = torch.tensor(cu, dtype=torch.int32, device=dev)
    q, k, v, table, lut, dout = (x[0] if x.dim() == 4 else x for x in make(dev, dtype, 1, T, T, H, Hk, D, fused=True, bidirectional=not causal))
    m = (torch.rand(T, generator=g) < 0.9).to(dev)
    for mask in (None, m):
        base = None
        for hint in (None, 1300, 64, 1):
            r = passes(q, k, v, table, lut, dout, cu_q=cut, cu_k=cut, max_q=hint, max_k=hint, causal=causal, key_mask=mask)
            base = base or r
            assert all(torch.equal(x, y) for x, y in zip(r, base)), hint
        total = torch.zeros(table.shape, dtype=F64, device=dev)
        for b, n in enumerate(lens):
            s = slice(cu[b], cu[b] + n)
            if n and (b % 20 == 0 or n > 100):
                one = passes(q[None, s], k[None, s], v[None, s], table, lut, dout[None, s], causal=causal, key_mask=None if mask is None else mask[None, s])
                for x, y in zip((base[0][s], base[1][:, s], base[2][s]), (one[0][0], one[1][0], one[2][0])):
                    assert torch.equal(x, y), b
                assert rel(base[3][s], one[3][0]) < TOL[dtype] and rel(base[4][s], one[4][0]) < TOL[dtype]
        for x in (base[0], base[2], base[3], base[4]):
            assert not x[:11].any() and not x[cu[-1]:].any()
        # dtable of every sequence for itself, in 64 bits
        for b, n in enumerate(lens):
            if n:
                s = slice(cu[b], cu[b] + n)
                total += passes(q[None, s], k[None, s], v[None, s], table.float(), lut, dout[None, s], causal=causal,
                                key_mask=None if mask is None else mask[None, s])[5].to(F64)
        assert rel(base[5], total) < 2 * TOL[dtype]


def test_packed_batch_of_many_sequences(dev):
    """2048 sequences in 131072 tokens without a hint"""
    B, n, H, D = 2048, 64, 12, 16
    q, k, v, table, lut, dout = make(dev, torch.bfloat16, B, n, n, H, H, D, fused=True)
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev) * n
    a = passes(q, k, v, table, lut, dout)
    free = torch.cuda.max_memory_allocated(dev)
    torch.cuda.reset_peak_memory_stats(dev)
    b = passes(*(x.flatten(0, 1) for x in (q, k, v)), table, lut, dout.flatten(0, 1), cu_q=cu, cu_k=cu)
    print("peak", free >> 20, torch.cuda.max_memory_allocated(dev) >> 20, flush=True)
    assert torch.equal(b[0], a[0].flatten(0, 1)) and all(torch.equal(b[i], a[i].flatten(0, 1)) for i in (2, 3, 4)) and rel(b[5], a[5]) < TOL[torch.bfloat16]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_sequence_into_given_outputs(dev, dtype):
    """offsets of no sequence, outputs given: nothing to launch, everything stays; and sequences of queries without keys, of keys without queries"""
    ops = _ops()
    q, k, v, table, lut, dout = (x[0] if x.dim() == 4 else x for x in make(dev, dtype, 1, 90, 90, 4, 2, 64))
    cu = torch.zeros(1, dtype=torch.int32, device=dev)
    mine = torch.full_like(q, 7.0)
    assert ops.relpos_attn_fwd(q, k, v, table, lut, cu_q=cu, cu_k=cu, out=mine)[0] is mine and bool((mine == 7).all())
    none, all_ = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 0, 0], [0, 50, 90]))
    for many in (False, True):                              # (two sequences, and more than 64)
        if many:
            none, all_ = none[:1].expand(101).contiguous(), torch.cat([all_[:1].expand(50), all_[1:2].expand(30), all_[2:].expand(21)]).contiguous()
        a = passes(q[:0], k, v, table, lut, dout[:0], cu_q=none, cu_k=all_)
        assert a[0].shape[0] == 0 and not a[3].any() and not a[4].any() and not a[5].any() and bool(torch.isfinite(a[5]).all())
        a = passes(q, k[:0], v[:0], table, lut, dout, cu_q=all_, cu_k=none)
        assert not a[0].any() and bool((a[1] == -math.inf).all()) and not a[2].any() and not a[5].any()


@pytest.mark.parametrize("seed", range(3))
def test_bad_offsets_of_many_sequences_stay_inside(dev, seed):
    """100 sequences whose offsets run backwards, past the buffers and below zero: clamped on the device, some rows are wrong, none outside is touched"""
    ops = _ops()
    T = 700
    q, k, v, table, lut, dout = (x[0] if x.dim() == 4 else x for x in make(dev, torch.bfloat16, 1, T, T, 4, 2, 64, seed=seed))
    g = torch.Generator().manual_seed(seed)
    cu = torch.randint(-300, T + 900, (101,), generator=g).int()
    cu[7], cu[50] = -(1 << 31), (1 << 31) - 1
    if seed:
        cu = cu.sort().values if seed == 1 else cu.sort(descending=True).values
    cu = cu.to(dev)
    guard = [torch.full((3 * T,) + x.shape[1:], 7.0, dtype=x.dtype, device=dev) for x in (q, q, k, v)]
    for causal in (False, True):
        _, lse = ops.relpos_attn_fwd(q, k, v, table, lut, cu_q=cu, cu_k=cu, out=guard[0][T:2 * T], causal=causal)
        lse = torch.nan_to_num(lse, neginf=0.0)
        dt = ops.relpos_attn_bwd(q, k, v, table, lut, torch.zeros_like(q), dout, lse, cu_q=cu, cu_k=cu, dq=guard[1][T:2 * T], dk=guard[2][T:2 * T], dv=guard[3][T:2 * T],
                                 causal=causal)[3]
        assert dt.shape == table.shape
        for x in guard:
            assert bool((x[:T] == 7).all()) and bool((x[2 * T:] == 7).all())


# ---- two 16-row tiles a wave (bf16), against the 64-bit oracle, dtable included
TWO = [  # B, Lq, Lk, H, Hk, D
    (12, 385, 385, 12, 12, 64), (20, 130, 130, 12, 12, 32), (40, 70, 70, 12, 12, 64), (8, 300, 300, 16, 16, 96), (8, 260, 411, 24, 12, 40), (5, 700, 700, 24, 12, 64),
    (26, 1100, 100, 12, 12, 64)]


def thresholds():
    """grids of up to so many workgroups of two tiles take one: forward and dQ at D <= 64, beyond, dK / dV"""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spokennlp_amd", "csrc", "relpos_launch.h")).read()
    wide, narrow = re.search(r"rp_qt\(rp_wgs_of_two\(a\), a\.D > 64 \? (\d+) : (\d+), dtype\)", text).groups()
    return int(narrow), int(wide), int(re.search(r"rp_qt\(rp_blocks_of_two\(a, a\.Lk, a\.Tk\) \* a\.kv_heads, (\d+), dtype\)", text).group(1))


@pytest.mark.parametrize("shape", TWO)
@pytest.mark.parametrize("how", ["plain", "causal", "ragged", "span 48", "span 200", "packed"])
def test_two_tiles_a_wave(dev, shape, how):
    """forward, dQ and (D <= 64) dK / dV with 32 rows a wave: whole and half empty blocks, blocks of few keys, heads dealt over workgroups, rows cut into pieces"""
    print("CASE", shape, how, flush=True)
    B, Lq, Lk, H, Hk, D = shape
    narrow, wide, kv = thresholds()
    assert -(-Lq // 128) * B * H > (narrow if D <= 64 else wide) and (D > 64 or -(-Lk // 128) * B * Hk > kv), "a shape for one tile"
    span = int(how[5:]) if how.startswith("span") else 128
    q, k, v, table, lut, dout = make(dev, torch.bfloat16, *shape, max_distance=span, bidirectional=how != "causal", fused=Lq == Lk)
    opt = {}
    if how == "causal":
        opt = dict(causal=True, align_end=Lq < Lk)
    elif how == "ragged":
        opt = dict(k_lens=torch.tensor([max(1, Lk - 31 * b) for b in range(B)], dtype=torch.int32, device=dev),
                   key_mask=torch.rand(B, Lk, generator=torch.Generator().manual_seed(4)).to(dev) < 0.8)
    a = check(dev, q, k, v, table, lut, dout, **opt)
    if how == "packed":
        cq, ck = (torch.arange(B + 1, dtype=torch.int32, device=dev) * n for n in (Lq, Lk))
        p = passes(*(x.flatten(0, 1) for x in (q, k, v)), table, lut, dout.flatten(0, 1), cu_q=cq, cu_k=ck)
        assert torch.equal(p[0], a[0].flatten(0, 1)) and torch.equal(p[1], a[1].transpose(0, 1).flatten(1)) and torch.equal(p[2], a[2].flatten(0, 1))
        assert rel(p[3], a[3].flatten(0, 1)) < TOL[torch.bfloat16] and rel(p[4], a[4].flatten(0, 1)) < TOL[torch.bfloat16] and rel(p[5], a[5]) < TOL[torch.bfloat16]


def test_spans_of_one_and_none_with_two_tiles(dev):
    """the diagonal sums where the near band is narrower than a tile: span 0 (one bucket: no positions), 1 and 15 with an unordered map"""
    ops = _ops()
    q, k, v, _, _, dout = make(dev, torch.bfloat16, 12, 385, 385, 12, 12, 64)
    table = torch.randn(5, 12, generator=torch.Generator().manual_seed(1)).to(dev)
    for span in (1, 15):
        lut = torch.randint(0, 5, (2 * span + 1,), generator=torch.Generator().manual_seed(span)).int().to(dev)
        check(dev, q, k, v, table, lut, dout, causal=span == 15)
    check(dev, q, k, v, table, torch.zeros(1, dtype=torch.int32, device=dev) + 2, dout, one_bucket=True)
    assert ops.relpos_bias_fwd(table, lut, 3, 3).shape == (12, 3, 3)
