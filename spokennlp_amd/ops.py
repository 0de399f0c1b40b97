"""Thin torch-tensor wrappers over the libamdseg C ABI (tensors are storage only: data_ptr + stream go to HIP).

Every function launches on torch's current HIP stream and raises ``AmdsegError`` on a non-zero return code.
"""
import ctypes as C

import torch

from . import lib as L
from .lib import BF16, F32, EPI_NONE, EPI_BIAS, EPI_BIAS_GELU, EPI_ADD_RES, EPI_GELU_BWD  # noqa: F401


def _s():
    return torch.cuda.current_stream().cuda_stream


def _p(t):
    return None if t is None else t.data_ptr()


def _dt(t):
    if t.dtype == torch.bfloat16:
        return BF16
    if t.dtype == torch.float32:
        return F32
    raise TypeError(f"unsupported dtype {t.dtype}")


def _chk(t, name):
    if not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous device tensor")


def gemm_nt(A, B, epilogue=EPI_NONE, bias=None, R=None, out=None, out2=None, out_dtype=torch.bfloat16):
    """C[M,N] = A[M,K] @ B[N,K]^T with fused epilogue; A, B bf16. Returns C (and C2 for EPI_BIAS_GELU)."""
    _chk(A, "A"); _chk(B, "B")
    M, K = A.shape
    N = B.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=A.device)
    if (epilogue & 0xff) == EPI_BIAS_GELU and out2 is None:
        out2 = torch.empty((M, N), dtype=torch.bfloat16, device=A.device)
    rc = L.load().amdseg_gemm_nt(_p(A), A.stride(0), _p(B), B.stride(0), _p(out), out.stride(0), M, N, K, epilogue,
                                 _p(bias), _p(R), 0 if R is None else R.stride(0), _p(out2),
                                 0 if out2 is None else out2.stride(0), 1 if out.dtype == torch.float32 else 0, _s())
    L.check(rc, "amdseg_gemm_nt")
    return (out, out2) if (epilogue & 0xff) == EPI_BIAS_GELU else out


def gemm_tn_grouped(As, Bs, Cs, accumulate=False, colsums=None):
    """For each i: Cs[i][N_i,K_i] (+)= As[i]^T @ Bs[i]  (As[i]: [M,N_i] bf16, Bs[i]: [M,K_i] bf16, Cs[i] fp32)."""
    n = len(As)
    M = As[0].shape[0]
    vpa = (C.c_void_p * n)(*[a.data_ptr() for a in As])
    vpb = (C.c_void_p * n)(*[b.data_ptr() for b in Bs])
    vpc = (C.c_void_p * n)(*[c.data_ptr() for c in Cs])
    ia = (C.c_int * n)(*[a.stride(0) for a in As])
    ib = (C.c_int * n)(*[b.stride(0) for b in Bs])
    ic = (C.c_int * n)(*[c.stride(0) for c in Cs])
    nn = (C.c_int * n)(*[a.shape[1] for a in As])
    kk = (C.c_int * n)(*[b.shape[1] for b in Bs])
    if colsums is None:
        rc = L.load().amdseg_gemm_tn_grouped(n, vpa, ia, vpb, ib, vpc, ic, nn, kk, M, 1 if accumulate else 0, _s())
        L.check(rc, "amdseg_gemm_tn_grouped")
        return Cs
    # bias gradients: colsums[i] (fp32 [N_i] or None) (+)= column sums of As[i]
    scratch = [None if c is None else torch.empty(max((M + 127) // 128, b.shape[1] // 128) * a.shape[1], dtype=torch.float32, device=a.device)
               for a, b, c in zip(As, Bs, colsums)]
    vpo = (C.c_void_p * n)(*[None if c is None else c.data_ptr() for c in colsums])
    vps = (C.c_void_p * n)(*[None if c is None else c.data_ptr() for c in scratch])
    rc = L.load().amdseg_gemm_tn_grouped_bias(n, vpa, ia, vpb, ib, vpc, ic, nn, kk, M, 1 if accumulate else 0, vpo, vps, _s())
    L.check(rc, "amdseg_gemm_tn_grouped_bias")
    return Cs


def attn_fwd(qkv, mask_bias, B, Lseq, heads, p=0.0, seed=0, need_lse=True, scale=0.125):
    H = heads * 64
    ctx = torch.empty((B * Lseq, H), dtype=torch.bfloat16, device=qkv.device)
    lse = torch.empty((B * heads * Lseq,), dtype=torch.float32, device=qkv.device) if need_lse else None
    rc = L.load().amdseg_attn_fwd(_p(qkv), _p(mask_bias), _p(ctx), _p(lse), B, Lseq, heads, scale, p, seed, _s())
    L.check(rc, "amdseg_attn_fwd")
    return ctx, lse


def attn_bwd(qkv, mask_bias, ctx, dctx, lse, B, Lseq, heads, p=0.0, seed=0, scale=0.125):
    dqkv = torch.empty_like(qkv)
    delta = torch.empty((B * heads * Lseq,), dtype=torch.float32, device=qkv.device)
    rc = L.load().amdseg_attn_bwd(_p(qkv), _p(mask_bias), _p(ctx), _p(dctx), _p(lse), _p(delta), _p(dqkv), B, Lseq, heads,
                                  scale, p, seed, _s())
    L.check(rc, "amdseg_attn_bwd")
    return dqkv


def attn_keepmask(B, Lseq, heads, p, seed, device, kend=None):
    """dropout keep masks of one attention layer (amdseg_attn_keepmask): uint8 buffer holding layout A then layout B"""
    lib = L.load()
    keep = torch.empty(lib.amdseg_attn_keepmask_bytes(B, Lseq, heads), dtype=torch.uint8, device=device)
    L.check(lib.amdseg_attn_keepmask(_p(keep), B, Lseq, heads, p, seed, _p(kend), _s()), "amdseg_attn_keepmask")
    return keep


def attn_fwd_keep(qkv, mask_bias, B, Lseq, heads, p, keep, need_lse=True, scale=0.125):
    H = heads * 64
    ctx = torch.empty((B * Lseq, H), dtype=torch.bfloat16, device=qkv.device)
    lse = torch.empty((B * heads * Lseq,), dtype=torch.float32, device=qkv.device) if need_lse else None
    L.check(L.load().amdseg_attn_fwd_keep(_p(qkv), _p(mask_bias), _p(ctx), _p(lse), B, Lseq, heads, scale, p, _p(keep), _s()), "amdseg_attn_fwd_keep")
    return ctx, lse


def attn_bwd_keep(qkv, mask_bias, ctx, dctx, lse, B, Lseq, heads, p, keep, scale=0.125):
    dqkv = torch.empty_like(qkv)
    delta = torch.empty((B * heads * Lseq,), dtype=torch.float32, device=qkv.device)
    L.check(L.load().amdseg_attn_bwd_keep(_p(qkv), _p(mask_bias), _p(ctx), _p(dctx), _p(lse), _p(delta), _p(dqkv), B, Lseq, heads,
                                          scale, p, _p(keep), _s()), "amdseg_attn_bwd_keep")
    return dqkv


def attn_keepmask_band(B, Lseq, heads, p, seed, window, nglobal, device):
    """keep masks of a band (Longformer) layer: same buffer layout as attn_keepmask, only the cells the band kernels visit are written"""
    lib = L.load()
    keep = torch.zeros(lib.amdseg_attn_keepmask_bytes(B, Lseq, heads), dtype=torch.uint8, device=device)
    L.check(lib.amdseg_attn_keepmask_band(_p(keep), B, Lseq, heads, p, seed, window, nglobal, _s()), "amdseg_attn_keepmask_band")
    return keep


def attn_band_fwd_keep(qkv, mask_bias, B, Lseq, heads, window, nglobal, p, keep, scale=0.125):
    ctx = torch.empty((B * Lseq, heads * 64), dtype=torch.bfloat16, device=qkv.device)
    lse = torch.empty((B * heads * Lseq,), dtype=torch.float32, device=qkv.device)
    L.check(L.load().amdseg_attn_band_fwd_keep(_p(qkv), _p(mask_bias), _p(ctx), _p(lse), B, Lseq, heads, scale, p, _p(keep), window, nglobal, _s()),
            "amdseg_attn_band_fwd_keep")
    return ctx, lse


def attn_band_bwd_keep(qkv, mask_bias, ctx, dctx, lse, B, Lseq, heads, window, nglobal, p, keep, scale=0.125):
    dqkv = torch.empty_like(qkv)
    delta = torch.empty((B * heads * Lseq,), dtype=torch.float32, device=qkv.device)
    L.check(L.load().amdseg_attn_band_bwd_keep(_p(qkv), _p(mask_bias), _p(ctx), _p(dctx), _p(lse), _p(delta), _p(dqkv), B, Lseq, heads, scale, p,
                                               _p(keep), window, nglobal, _s()), "amdseg_attn_band_bwd_keep")
    return dqkv


def attn_list_fwd(qkv, mask_bias, B, Lseq, heads, klist, kcnt, stride, ctx=None, lse=None, scale=0.125, korder=None):
    """BigBird block-list attention (amdseg_attn_list_fwd); klist/kcnt: int32 device tensors [heads, L/64, stride] / [heads, L/64]"""
    H = heads * 64
    if ctx is None:
        ctx = torch.empty((B * Lseq, H), dtype=torch.bfloat16, device=qkv.device)
    if lse is None:
        lse = torch.empty((B * heads * Lseq,), dtype=torch.float32, device=qkv.device)
    rc = L.load().amdseg_attn_list_fwd(_p(qkv), _p(mask_bias), _p(ctx), _p(lse), B, Lseq, heads, scale, _p(klist), _p(kcnt), stride, _p(korder), _s())
    L.check(rc, "amdseg_attn_list_fwd")
    return ctx, lse


def attn_list_f32(qkv, mask_bias, B, Lseq, heads, klist, kcnt, stride, ctx=None, scale=0.125):
    """fp32 parity-mode block-list attention (amdseg_attn_list_f32): qkv fp32 [B*L, 3*heads*64] -> ctx fp32 [B*L, heads*64]"""
    if ctx is None:
        ctx = torch.empty((B * Lseq, heads * 64), dtype=torch.float32, device=qkv.device)
    rc = L.load().amdseg_attn_list_f32(_p(qkv), _p(mask_bias), _p(ctx), B, Lseq, heads, scale, _p(klist), _p(kcnt), stride, _s())
    L.check(rc, "amdseg_attn_list_f32")
    return ctx


def attn_list_bwd(qkv, mask_bias, ctx, dctx, lse, B, Lseq, heads, klist, kcnt, qlist, qcnt, stride, dqkv=None, delta=None, scale=0.125,
                  korder=None, qorder=None):
    if dqkv is None:
        dqkv = torch.empty_like(qkv)
    if delta is None:
        delta = torch.empty((B * heads * Lseq,), dtype=torch.float32, device=qkv.device)
    rc = L.load().amdseg_attn_list_bwd(_p(qkv), _p(mask_bias), _p(ctx), _p(dctx), _p(lse), _p(delta), _p(dqkv), B, Lseq, heads, scale,
                                       _p(klist), _p(kcnt), _p(qlist), _p(qcnt), stride, _p(korder), _p(qorder), _s())
    L.check(rc, "amdseg_attn_list_bwd")
    return dqkv


def attn_band_fwd(qkv, mask_bias, B, Lseq, heads, window, nglobal=1, p=0.0, seed=0, need_lse=True, scale=0.125):
    H = heads * 64
    ctx = torch.empty((B * Lseq, H), dtype=torch.bfloat16, device=qkv.device)
    lse = torch.empty((B * heads * Lseq,), dtype=torch.float32, device=qkv.device) if need_lse else None
    rc = L.load().amdseg_attn_band_fwd(_p(qkv), _p(mask_bias), _p(ctx), _p(lse), B, Lseq, heads, scale, p, seed, window, nglobal, _s())
    L.check(rc, "amdseg_attn_band_fwd")
    return ctx, lse


def attn_band_bwd(qkv, mask_bias, ctx, dctx, lse, B, Lseq, heads, window, nglobal=1, p=0.0, seed=0, scale=0.125):
    dqkv = torch.empty_like(qkv)
    delta = torch.empty((B * heads * Lseq,), dtype=torch.float32, device=qkv.device)
    rc = L.load().amdseg_attn_band_bwd(_p(qkv), _p(mask_bias), _p(ctx), _p(dctx), _p(lse), _p(delta), _p(dqkv), B, Lseq, heads,
                                       scale, p, seed, window, nglobal, _s())
    L.check(rc, "amdseg_attn_band_bwd")
    return dqkv


def attn_band_f32(qkv, mask_bias, B, Lseq, heads, window, nglobal=1, scale=0.125):
    ctx = torch.empty((B * Lseq, heads * 64), dtype=torch.float32, device=qkv.device)
    rc = L.load().amdseg_attn_band_f32(_p(qkv), _p(mask_bias), _p(ctx), B, Lseq, heads, scale, window, nglobal, _s())
    L.check(rc, "amdseg_attn_band_f32")
    return ctx


# ---- Longformer global row (csrc/longformer.hip): x [B*L, H] bf16/fp32; vec [B, heads, H] fp32; planes [B, heads, L] fp32
def lf_rowvec_dot(x, vec, B, Lseq, add_tok=None, add_bh=None):
    """x: [B*L, H] (rows may be strided: a column block of a wider matrix)"""
    heads, H = vec.shape[1], vec.shape[2]
    out = torch.empty((B, heads, Lseq), dtype=torch.float32, device=x.device)
    rc = L.load().amdseg_lf_rowvec_dot_ld(_p(x), x.stride(0), _p(vec), _p(add_tok), _p(add_bh), _p(out), B, Lseq, H, heads, _dt(x), _s())
    L.check(rc, "amdseg_lf_rowvec_dot_ld")
    return out


def lf_softmax_fwd(scores, p=0.0, seed=0):
    """scores [B, heads, L] fp32 is overwritten with the probabilities; returns (p, dropped p, sum of dropped p [B, heads])."""
    B, heads, Lseq = scores.shape
    pd = torch.empty_like(scores)
    sp = torch.empty((B, heads), dtype=torch.float32, device=scores.device)
    rc = L.load().amdseg_lf_softmax_fwd(_p(scores), _p(pd), _p(sp), B * heads, Lseq, p, seed, _s())
    L.check(rc, "amdseg_lf_softmax_fwd")
    return scores, pd, sp


def lf_softmax_bwd(p_saved, dpd, p=0.0, seed=0):
    """dpd is overwritten with ds; returns (ds, recomputed dropped p)."""
    B, heads, Lseq = p_saved.shape
    pd = torch.empty_like(p_saved)
    rc = L.load().amdseg_lf_softmax_bwd(_p(p_saved), _p(dpd), _p(pd), B * heads, Lseq, p, seed, _s())
    L.check(rc, "amdseg_lf_softmax_bwd")
    return dpd, pd


def lf_wsum(x, coef, H, partials=None):
    B, heads, Lseq = coef.shape
    if partials is None:
        partials = torch.empty((B * (Lseq // 64) * heads * H,), dtype=torch.float32, device=x.device)
    y = torch.empty((B, heads, H), dtype=torch.float32, device=x.device)
    rc = L.load().amdseg_lf_wsum_ld(_p(x), x.stride(0), _p(coef), _p(partials), _p(y), B, Lseq, H, heads, _dt(x), _s())
    L.check(rc, "amdseg_lf_wsum_ld")
    return y


def lf_dx_update(dx, coefA, vecA, coefB, vecB, vt_ws=None, assign=False):
    """dx: [B*L, H] rows (may be strided); assign=True overwrites instead of accumulating"""
    B, heads, Lseq = coefA.shape
    H = vecA.shape[2]
    if vt_ws is None and dx.dtype == torch.bfloat16:
        vt_ws = torch.empty(B * H * 32, dtype=torch.bfloat16, device=dx.device)
    rc = L.load().amdseg_lf_dx_update_ld(_p(dx), dx.stride(0), 1 if assign else 0, _p(coefA), _p(vecA), _p(coefB), _p(vecB), _p(vt_ws),
                                         B, Lseq, H, heads, _dt(dx), _s())
    L.check(rc, "amdseg_lf_dx_update_ld")


# ---- PoNet token mixing (csrc/ponet.hip, csrc/ponet_global.hip)
def ponet_global_scratch(B, Lseq, H, heads, device):
    return torch.empty(int(L.load().amdseg_ponet_global_scratch_floats(B, Lseq, H, heads)), dtype=torch.float32, device=device)


def ponet_global_fwd(hq, hk, coef_mean, mask_bias, B, Lseq, H, heads, p=0.0, seed=0, scratch=None):
    """hq, hk: bf16 column blocks [B*L, H] of the projection (same row stride).  Returns (g [B,H], vecq [B,H], scores [B,heads,L], lse [B,heads])."""
    dev = hk.device
    if scratch is None:
        scratch = ponet_global_scratch(B, Lseq, H, heads, dev)
    f = dict(dtype=torch.float32, device=dev)
    vecq, g = torch.empty(B, H, **f), torch.empty(B, H, **f)
    scores, lse = torch.empty(B, heads, Lseq, **f), torch.empty(B, heads, **f)
    assert hq.stride(0) == hk.stride(0)
    rc = L.load().amdseg_ponet_global_fwd(_p(hq), _p(hk), hk.stride(0), _p(coef_mean), _p(mask_bias), B, Lseq, H, heads, p, seed, _p(scratch),
                                          _p(vecq), _p(scores), _p(lse), _p(g), _s())
    L.check(rc, "amdseg_ponet_global_fwd")
    return g, vecq, scores, lse


def ponet_global_bwd(hk, coef_mean, vecq, scores, lse, dg, dhq, dhk, B, Lseq, H, heads, p=0.0, seed=0, scratch=None, dpd_ws=None):
    """writes the dHq / dHk column blocks (bf16, same row stride) of the projection gradient"""
    dev = hk.device
    if scratch is None:
        scratch = ponet_global_scratch(B, Lseq, H, heads, dev)
    if dpd_ws is None:
        dpd_ws = torch.empty(B, heads, Lseq, dtype=torch.float32, device=dev)
    assert dhq.stride(0) == dhk.stride(0)
    rc = L.load().amdseg_ponet_global_bwd(_p(hk), hk.stride(0), _p(coef_mean), _p(vecq), _p(scores), _p(lse), _p(dg), B, Lseq, H, heads, p, seed,
                                          _p(scratch), _p(dpd_ws), _p(dhq), _p(dhk), dhk.stride(0), _s())
    L.check(rc, "amdseg_ponet_global_bwd")


def ponet_plan(mask_bias, run_start, B, Lseq):
    """work lists of the PoNet pooling kernels for one batch (csrc/ponet.hip): int32 [2 + 2*B*L] on the device, no host sync"""
    work = torch.empty(2 + 2 * B * Lseq, dtype=torch.int32, device=mask_bias.device)
    rc = L.load().amdseg_ponet_plan(_p(mask_bias), _p(run_start), _p(work), B, Lseq, _s())
    L.check(rc, "amdseg_ponet_plan")
    return work


def ponet_pool_fwd(proj, mask_bias, run_start, run_end, work, g, part, parg, ctx, B, Lseq, H):
    rc = L.load().amdseg_ponet_pool_fwd(_p(proj), proj.stride(0), _p(mask_bias), _p(run_start), _p(run_end), _p(work), _p(g), _p(part),
                                        _p(parg), _p(ctx), B, Lseq, H, _s())
    L.check(rc, "amdseg_ponet_pool_fwd")


def ponet_pool_bwd(proj, mask_bias, run_start, run_end, work, g, part, parg, dctx, dproj, psum, B, Lseq, H):
    """returns dg [B, H] fp32: the per-sequence sum of dctx * Ho over the valid tokens (gradient of the global aggregate)"""
    dg = torch.empty(B, H, dtype=torch.float32, device=proj.device)
    rc = L.load().amdseg_ponet_pool_bwd(_p(proj), proj.stride(0), _p(mask_bias), _p(run_start), _p(run_end), _p(work), _p(g), _p(part),
                                        _p(parg), _p(dctx), _p(dproj), _p(dg), _p(psum), B, Lseq, H, _s())
    L.check(rc, "amdseg_ponet_pool_bwd")
    return dg


def embed_ln_fwd(ids, type_ids, pos_ids, word, pos, typ, gamma, beta, Lseq, eps, p=0.0, seed=0, dtype=torch.bfloat16,
                 save=True):
    M = ids.numel()
    H = word.shape[1]
    dev = word.device
    out = torch.empty((M, H), dtype=dtype, device=dev)
    z = torch.empty((M, H), dtype=dtype, device=dev) if save else None
    mean = torch.empty((M,), dtype=torch.float32, device=dev) if save else None
    rstd = torch.empty((M,), dtype=torch.float32, device=dev) if save else None
    rc = L.load().amdseg_embed_ln_fwd(_p(ids), _p(type_ids), _p(pos_ids), _p(word), _p(pos), _p(typ), _p(gamma), _p(beta),
                                      _p(z), _p(out), _p(mean), _p(rstd), M, Lseq, H, word.shape[0], typ.shape[0],
                                      pos.shape[0], eps, p, seed, _dt(out), _s())
    L.check(rc, "amdseg_embed_ln_fwd")
    return out, z, mean, rstd


def embed_bwd(dz, ids, type_ids, pos_ids, dword, dpos, dtyp, Lseq, pad_id=-1, type0_holds_colsum=False):
    """type0_holds_colsum: row 0 of dtyp already holds the column sum of dz (include/amdseg.h: type_vocab < 0)"""
    M, H = dz.shape
    rc = L.load().amdseg_embed_bwd(_p(dz), _p(ids), _p(type_ids), _p(pos_ids), _p(dword), _p(dpos), _p(dtyp), M, Lseq, H,
                                   dword.shape[0], -dtyp.shape[0] if type0_holds_colsum else dtyp.shape[0], dpos.shape[0], pad_id,
                                   _dt(dz), _s())
    L.check(rc, "amdseg_embed_bwd")


def add_ln_fwd(y, resid, gamma, beta, eps, p=0.0, seed=0):
    """y is overwritten with z = resid + dropout(y); returns (out, mean, rstd)."""
    M, H = y.shape
    out = torch.empty_like(y)
    mean = torch.empty((M,), dtype=torch.float32, device=y.device)
    rstd = torch.empty((M,), dtype=torch.float32, device=y.device)
    rc = L.load().amdseg_add_ln_fwd(_p(y), _p(resid), _p(gamma), _p(beta), _p(out), _p(mean), _p(rstd), M, H, eps, p, seed,
                                    _dt(y), _s())
    L.check(rc, "amdseg_add_ln_fwd")
    return out, mean, rstd


def add_ln_fwd_keepmask(y, resid, gamma, beta, eps, p, seed, B, Lseq, heads, p_attn, seed_attn, kend=None, window=0, nglobal=0, drop_bits=None,
                        keep_z=True):
    """add_ln_fwd AND the keep masks of an attention layer as one launch (amdseg_add_ln_fwd_keepmask); returns (out, mean, rstd, keep)"""
    M, H = y.shape
    lib = L.load()
    out = torch.empty_like(y)
    mean = torch.empty((M,), dtype=torch.float32, device=y.device)
    rstd = torch.empty((M,), dtype=torch.float32, device=y.device)
    mk = torch.zeros if window > 0 else torch.empty
    keep = mk(lib.amdseg_attn_keepmask_bytes(B, Lseq, heads), dtype=torch.uint8, device=y.device)
    rc = lib.amdseg_add_ln_fwd_keepmask(_p(y), _p(resid), _p(gamma), _p(beta), _p(out), _p(mean), _p(rstd), M, H, eps, p, seed, _dt(y),
                                        _p(drop_bits), 1 if keep_z else 0, _p(keep), B, Lseq, heads, p_attn, seed_attn, _p(kend), window, nglobal, _s())
    L.check(rc, "amdseg_add_ln_fwd_keepmask")
    return out, mean, rstd, keep


LNB_ROWS = 16      # rows per workgroup of ln_bwd / rowdot_bwd (csrc/elementwise.hip)


def ln_partials_numel(M, H):
    return 3 * ((M + LNB_ROWS - 1) // LNB_ROWS) * H


def ln_bwd(dy, z, mean, rstd, gamma, p=0.0, seed=0, dgamma=None, dbeta=None, dbias=None, accumulate=False, partials=None):
    M, H = dy.shape
    dz = torch.empty_like(dy)
    dbr = torch.empty_like(dy) if p > 0 else None
    if partials is None and (dgamma is not None or dbeta is not None or dbias is not None):
        partials = torch.empty((ln_partials_numel(M, H),), dtype=torch.float32, device=dy.device)
    rc = L.load().amdseg_ln_bwd(_p(dy), _p(z), _p(mean), _p(rstd), _p(gamma), _p(dz), _p(dbr), _p(partials), _p(dgamma),
                                _p(dbeta), _p(dbias), M, H, p, seed, 1 if accumulate else 0, _dt(dy), _s())
    L.check(rc, "amdseg_ln_bwd")
    return dz, (dbr if dbr is not None else dz)


def colsum(x, out=None, accumulate=False, ncols=None):
    M = x.shape[0]
    N = ncols or x.shape[1]
    if out is None:
        out = torch.zeros((N,), dtype=torch.float32, device=x.device)
    partials = torch.empty((((M + 127) // 128) * N,), dtype=torch.float32, device=x.device)
    rc = L.load().amdseg_colsum(_p(x), x.stride(0), _p(partials), _p(out), M, N, 1 if accumulate else 0, _dt(x), _s())
    L.check(rc, "amdseg_colsum")
    return out


def dropout(x, p, seed, out_dtype=None):
    y = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    rc = L.load().amdseg_dropout(_p(x), _p(y), x.numel(), p, seed, _dt(x), _dt(y), _s())
    L.check(rc, "amdseg_dropout")
    return y


def cast(x, dtype):
    y = torch.empty(x.shape, dtype=dtype, device=x.device)
    rc = L.load().amdseg_cast(_p(x), _p(y), x.numel(), _dt(x), _dt(y), _s())
    L.check(rc, "amdseg_cast")
    return y


def cast_transpose(W, Wb=None, Wt=None):
    N, K = W.shape
    rc = L.load().amdseg_cast_transpose(_p(W), _p(Wb), _p(Wt), N, K, _s())
    L.check(rc, "amdseg_cast_transpose")


def rowdot_fwd(x, W, b):
    M, H = x.shape
    Cc = W.shape[0]
    out = torch.empty((M, Cc), dtype=torch.float32, device=x.device)
    rc = L.load().amdseg_rowdot_fwd(_p(x), _p(W), _p(b), _p(out), M, H, Cc, _dt(x), _s())
    L.check(rc, "amdseg_rowdot_fwd")
    return out


def rowdot_bwd(x, W, dlogits, dW=None, db=None, need_dx=True, accumulate=False):
    M, H = x.shape
    Cc = W.shape[0]
    dx = torch.empty_like(x) if need_dx else None
    partials = None
    if dW is not None or db is not None:
        partials = torch.empty((((M + LNB_ROWS - 1) // LNB_ROWS) * (Cc * H + Cc),), dtype=torch.float32, device=x.device)
    rc = L.load().amdseg_rowdot_bwd(_p(x), _p(W), _p(dlogits), _p(dx), _p(partials), _p(dW), _p(db), M, H, Cc,
                                    1 if accumulate else 0, _dt(x), _s())
    L.check(rc, "amdseg_rowdot_bwd")
    return dx


def adamw(p, g, m, v, shadow, lr, beta1, beta2, eps, wd, step, gscale=None, zero_grad=False, chunk_flags=None):
    rc = L.load().amdseg_adamw(_p(p), _p(g), _p(m), _p(v), _p(shadow), p.numel(), lr, beta1, beta2, eps, wd, step,
                               _p(gscale), 1 if zero_grad else 0, _p(chunk_flags), _s())
    L.check(rc, "amdseg_adamw")


def sumsq(x, out, partials, accumulate=False):
    rc = L.load().amdseg_sumsq(_p(x), x.numel(), _p(partials), _p(out), 1 if accumulate else 0, _s())
    L.check(rc, "amdseg_sumsq")


def clip_coef(sumsq_t, max_norm, extra_scale, coef, norm=None):
    rc = L.load().amdseg_clip_coef(_p(sumsq_t), max_norm, extra_scale, _p(coef), _p(norm), _s())
    L.check(rc, "amdseg_clip_coef")


def scale_(x, coef):
    rc = L.load().amdseg_scale(_p(x), x.numel(), _p(coef), _s())
    L.check(rc, "amdseg_scale")


def split3(x, out, order=0):
    """fp32 [M, K] -> bf16 [M, 3K] split image ([hi | hi | lo] for order 0, [hi | lo | hi] for order 1); csrc/parity.hip"""
    M, K = x.shape
    rc = L.load().amdseg_split3(_p(x), x.stride(0), _p(out), M, K, order, _s())
    L.check(rc, "amdseg_split3")
    return out


def split3_transpose(W, out):
    N, K = W.shape
    rc = L.load().amdseg_split3_transpose(_p(W), _p(out), N, K, _s())
    L.check(rc, "amdseg_split3_transpose")
    return out


def sattn_fwd(qkv, mask_bias, B, Lq, heads, p=0.0, keep=None, window=0, nglobal=0):
    """"parity" precision attention on split-bf16 products (amdseg_sattn_fwd): qkv fp32 [B*L, 3H] -> (ctx fp32, lse, the split image)"""
    H = heads * 64
    qs = split3(qkv, torch.empty(B * Lq, 9 * H, dtype=torch.bfloat16, device=qkv.device))
    ctx = torch.empty(B * Lq, H, dtype=torch.float32, device=qkv.device)
    lse = torch.empty(B * heads * Lq, dtype=torch.float32, device=qkv.device)
    L.check(L.load().amdseg_sattn_fwd(_p(qs), 9 * H, 6 * H, _p(mask_bias), _p(ctx), _p(lse), B, Lq, heads, 0.125, p, _p(keep), window, nglobal, _s()),
            "amdseg_sattn_fwd")
    return ctx, lse, qs


def sattn_bwd(qs, mask_bias, ctx, dctx, lse, B, Lq, heads, p=0.0, keep=None, window=0, nglobal=0):
    H = heads * 64
    dos = split3(dctx, torch.empty(B * Lq, 3 * H, dtype=torch.bfloat16, device=dctx.device))
    dqkv = torch.empty(B * Lq, 3 * H, dtype=torch.float32, device=dctx.device)
    delta = torch.empty_like(lse)
    L.check(L.load().amdseg_sattn_bwd(_p(qs), 9 * H, 6 * H, _p(mask_bias), _p(ctx), _p(dos), 3 * H, 2 * H, _p(lse), _p(delta), _p(dqkv), B, Lq,
                                      heads, 0.125, p, _p(keep), window, nglobal, _s()), "amdseg_sattn_bwd")
    return dqkv


def pattn_fwd(qkv, mask_bias, B, Lq, heads, p=0.0, seed=0):
    H = heads * 64
    ctx = torch.empty(B * Lq, H, dtype=torch.float32, device=qkv.device)
    lse = torch.empty(B * heads * Lq, dtype=torch.float32, device=qkv.device)
    rc = L.load().amdseg_pattn_fwd(_p(qkv), _p(mask_bias), _p(ctx), _p(lse), B, Lq, heads, 0.125, p, seed, _s())
    L.check(rc, "amdseg_pattn_fwd")
    return ctx, lse


def pattn_bwd(qkv, mask_bias, ctx, dctx, lse, B, Lq, heads, p=0.0, seed=0):
    dqkv = torch.empty_like(qkv)
    delta = torch.empty_like(lse)
    rc = L.load().amdseg_pattn_bwd(_p(qkv), _p(mask_bias), _p(ctx), _p(dctx), _p(lse), _p(delta), _p(dqkv), B, Lq, heads, 0.125, p, seed, _s())
    L.check(rc, "amdseg_pattn_bwd")
    return dqkv


# ---- attention under a learned relative position bias (csrc/relpos_fwd.hip, relpos_bwd.hip, relpos_bias.hip)
def relpos_bucket_list(num_buckets=32, max_distance=128, bidirectional=True):
    """bucket of rel = -max_distance .. max_distance (key position - query position) as a list of 2 * max_distance + 1 ints.  Half of a side's
    buckets hold one distance each, the others steps that grow with the distance up to max_distance; two sides, or (bidirectional=False) one: keys behind
    the query share bucket 0 with distance 0.  Distances are compared as whole numbers (n >= m (M / m)^(k / steps)  <=>  n^steps >= m^(steps - k) M^k), so
    no rounding of a logarithm moves one over a bucket's edge."""
    half = num_buckets // 2 if bidirectional else num_buckets
    m = half // 2
    steps = half - m
    if num_buckets < 1 or m < 1 or max_distance <= m:
        raise ValueError(f"num_buckets = {num_buckets}, max_distance = {max_distance}: a side needs two buckets and max_distance beyond its first half")
    near, k = list(range(m)), 0
    for n in range(m, max_distance + 1):
        while k + 1 < steps and n ** steps >= m ** (steps - k - 1) * max_distance ** (k + 1):
            k += 1
        near.append(m + k)
    if bidirectional:
        return near[:0:-1] + [near[0]] + [half + b for b in near[1:]]
    return near[:0:-1] + [near[0]] * (max_distance + 1)


def relpos_bucket_map(num_buckets=32, max_distance=128, bidirectional=True, device="cuda"):
    """relpos_bucket_list as the device tensor that the relpos_* functions take (build it once per model)"""
    return torch.tensor(relpos_bucket_list(num_buckets, max_distance, bidirectional), dtype=torch.int32, device=device)


def _rp_strides(t, name, esize):
    """element strides (sequence, row, head) of [B, L, heads, D] or packed [T, heads, D]"""
    st = t.stride()
    if t.numel() and st[-1] != 1 and t.shape[-1] != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous, strides are {st}")
    st = [0 if n == 1 else s for n, s in zip(t.shape[:-1], st[:-1])]
    if (t.data_ptr() | (st[-1] * esize) | (st[-2] * esize) | (st[0] * esize)) & 15:
        raise ValueError(f"{name}: rows must start on 16 bytes (strides {t.stride()}, element size {esize})")
    if not 0 <= st[-2] * esize <= 1 << 24:
        raise ValueError(f"{name}: rows at most 16 MiB apart (strides {t.stride()}, element size {esize})")
    return (st[0] if len(st) == 3 else 0, st[-2], st[-1])


def _rp_int(t, name, n, dev):
    if t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} elements on {dev}")
    return t.data_ptr()


def _rp_table(c, table, bucket_map, heads):
    if table.dim() != 2 or table.shape[1] != heads or table.shape[0] < 1 or not table.is_contiguous():
        raise ValueError(f"table must be a contiguous [buckets, {heads}] tensor, not {tuple(table.shape)}")
    n = bucket_map.numel()
    if n % 2 == 0 or n > 2049:
        raise ValueError(f"bucket_map must hold 2 * span + 1 entries with span <= 1024, not {n}")
    c.span, c.table_dtype, c.buckets = n // 2, _dt(table), table.shape[0]


def _rp_cfg(q, k, v, table, bucket_map, scale, key_mask, k_lens, cu_q, cu_k, max_q, max_k, causal, align_end, more_key, more):
    """-> (RelposCfg, shape of lse, workspace bytes forward, backward).  What follows from shapes, strides, types and options alone is worked out once per
    such combination and copied (a call on a few rows is otherwise longer on the host than on the GPU); pointers and devices are looked at every time.
    `more(c, shape of lse)` fills in the other tensors' strides, `more_key` is all that it looks at."""
    key = (q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(), q.dtype, k.dtype, v.dtype, table.shape, table.stride(), table.dtype, bucket_map.shape,
           bucket_map.stride(), bucket_map.dtype, scale if scale is None else float(scale), max_q if max_q is None else int(max_q),
           max_k if max_k is None else int(max_k), bool(causal), bool(align_end), cu_q is None or cu_q.shape, cu_k is None or cu_k.shape,
           k_lens is None, None if key_mask is None else (key_mask.shape, key_mask.stride(), key_mask.dtype), more_key)
    known = _rp_known.get(key)
    if known is None:
        known = _rp_plan(q, k, v, table, bucket_map, scale, key_mask, k_lens, cu_q, cu_k, max_q, max_k, causal, align_end, more)
        if len(_rp_known) >= 256:
            _rp_known.clear()
        _rp_known[key] = known
    c = L.RelposCfg.from_buffer_copy(known[0])
    dev = q.device
    if dev.type != "cuda" or k.device != dev or v.device != dev:
        raise ValueError("q, k, v must be on one GPU")
    if (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        raise ValueError("q, k, v: rows must start on 16 bytes")
    if table.device != dev or bucket_map.device != dev:
        raise ValueError(f"table and bucket_map must be on {dev}")
    c.table, c.map = table.data_ptr(), bucket_map.data_ptr()
    if cu_q is not None:
        c.cu_q, c.cu_k = _rp_int(cu_q, "cu_q", c.B + 1, dev), _rp_int(cu_k, "cu_k", c.B + 1, dev)
    if k_lens is not None:
        c.k_lens = _rp_int(k_lens, "k_lens", c.B, dev)
    if key_mask is not None:
        if key_mask.device != dev:
            raise ValueError(f"key_mask must be on {dev}")
        c.key_mask = key_mask.data_ptr()
    return c, known[1], known[2], known[3]


_rp_known = {}


def _rp_plan(q, k, v, table, bucket_map, scale, key_mask, k_lens, cu_q, cu_k, max_q, max_k, causal, align_end, more):
    """the checks and the part of RelposCfg that depend on no pointer"""
    packed = cu_q is not None
    if packed != (cu_k is not None):
        raise ValueError("cu_q and cu_k come together")
    nd = 3 if packed else 4
    if q.dim() != nd or k.dim() != nd or v.shape != k.shape:
        raise ValueError(f"q, k, v must be {'[tokens, heads, D]' if packed else '[B, L, heads, D]'}, not {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    c = L.RelposCfg()
    c.dtype = _dt(q)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k, v must share a dtype, not {q.dtype}, {k.dtype}, {v.dtype}")
    heads, D = q.shape[-2:]
    kv_heads = k.shape[-2]
    if k.shape[-1] != D or D < 8 or D > 128 or D % 8:
        raise ValueError(f"head dimension {D} (keys: {k.shape[-1]}): a multiple of 8 up to 128, the same for q, k, v")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads are no multiple of {kv_heads} key / value heads")
    c.heads, c.kv_heads, c.D = heads, kv_heads, D
    es = q.element_size()
    c.q_stride[:] = _rp_strides(q, "q", es)
    c.k_stride[:] = _rp_strides(k, "k", es)
    c.v_stride[:] = _rp_strides(v, "v", es)
    if packed:
        if k_lens is not None:
            raise ValueError("k_lens belongs to the padded form; packed sequences have cu_k")
        c.B, c.Tq, c.Tk = cu_q.numel() - 1, q.shape[0], k.shape[0]
        if c.B < 0:
            raise ValueError("cu_q needs at least one element")
        for n in (max_q, max_k):
            if n is not None and n < 0:
                raise ValueError("max_q / max_k must not be negative")
        c.Lq = max(1, min(c.Tq, c.Tq if max_q is None else int(max_q)))
        c.Lk = max(1, min(c.Tk, c.Tk if max_k is None else int(max_k)))
    else:
        if k.shape[0] != q.shape[0]:
            raise ValueError(f"q holds {q.shape[0]} sequences, k {k.shape[0]}")
        c.B, c.Lq, c.Lk = q.shape[0], q.shape[1], k.shape[1]
    if key_mask is not None:
        want = (c.Tk,) if packed else (c.B, c.Lk)
        if key_mask.dtype not in (torch.bool, torch.uint8) or tuple(key_mask.shape) != want:
            raise ValueError(f"key_mask must be a bool or uint8 tensor {want}, not {key_mask.dtype} {tuple(key_mask.shape)}")
        if key_mask.numel() and key_mask.shape[-1] > 1 and key_mask.stride(-1) != 1:
            raise ValueError("key_mask: the last dimension must be contiguous")
        c.mask_stride = 0 if packed or key_mask.shape[0] == 1 else key_mask.stride(0)
    _rp_table(c, table, bucket_map, heads)
    _rp_int(bucket_map, "bucket_map", 2 * c.span + 1, bucket_map.device)
    c.scale = D ** -0.5 if scale is None else float(scale)
    if not 1e-6 < c.scale < 1e6:
        raise ValueError(f"scale = {scale}: a positive number")
    c.causal, c.align_end = int(bool(causal)), int(bool(align_end))
    lse_shape = (heads, c.Tq) if packed else (c.B, heads, c.Lq)
    more(c, lse_shape)
    # the library sizes its workspaces from shapes; the two pointers it asks for (and whether there is a mask or offsets at all) stand in
    probe = L.RelposCfg.from_buffer_copy(c)
    probe.map = probe.table = 256
    if packed:
        probe.cu_q = probe.cu_k = 256
    lib = L.load()
    return (bytes(c), lse_shape, lib.amdseg_relpos_attn_ws_bytes(C.byref(probe), 0),
            lib.amdseg_relpos_attn_ws_bytes(C.byref(probe), 1))


def _rp_out(t, like, name, es):
    """a caller's output tensor: shape, dtype, and no two elements in one place"""
    if t.shape != like.shape or t.dtype != like.dtype:
        raise ValueError(f"{name} must be {tuple(like.shape)} {like.dtype}")
    at = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < at:
            raise ValueError(f"{name}: elements overlap (strides {t.stride()})")
        at = s * n if s * n > at else at
    return _rp_strides(t, name, es)


def _rp_dense(shape):
    """element strides (sequence, row, head) of a contiguous tensor"""
    st = [shape[-1] * shape[-2], shape[-1]]
    return (st[0] * shape[1] if len(shape) == 4 else 0, *st)


def _rp_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _rp_here(dev):
    """is a call's GPU the current one?  (If not, the call enters again under torch.cuda.device.)"""
    return torch._C._cuda_getDevice() == dev.index


def _rp_s(dev):
    """handle of the current stream of a GPU, without the Stream object (1 us less per call)"""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def relpos_attn_fwd(q, k, v, table, bucket_map, scale=None, key_mask=None, k_lens=None, cu_q=None, cu_k=None, max_q=None, max_k=None, causal=False,
                    align_end=False, need_lse=True, out=None):
    """softmax(scale q k^T + table[bucket_map[clamp(rel) + span]]) v with rel = key position - query position (amdseg_relpos_attn_fwd).

    Padded: q [B, Lq, heads, D], k / v [B, Lk, kv_heads, D] (any strides with a contiguous last dimension and rows on 16 bytes: column blocks of a fused
    projection, a cache), k_lens int32 [B] = keys held, key_mask bool / uint8 [B, Lk].  Packed: q [tokens, heads, D], cu_q / cu_k int32 [B + 1],
    max_q / max_k = longest sequence (hints that change no result; max_k saves time with a key mask), key_mask [tokens].  bf16 or fp32; table [buckets, heads] of either; scale: D ** -0.5.
    Query i stands at position i, or (align_end) so that the last query stands at the last key.  A row that sees no key: zero, lse -inf, no gradient.
    K / V rows that no query sees (masked, behind the keys held, with causal behind the last query) and q / dout of rows that see no key may hold anything;
    finite table entries may have any size (include/amdseg.h says how large ones count).
    Returns (out, lse); lse fp32 [B, heads, Lq] / [heads, tokens], None unless need_lse.  `out`: rows outside every packed sequence are left as they were
    (a fresh tensor has zeros there)."""
    def more(c, _):
        c.zero_tail = int(out is None)
        c.out_stride[:] = _rp_dense(q.shape) if out is None else _rp_out(out, q, "out", q.element_size())

    c, lse_shape, ws_bytes, _ = _rp_cfg(q, k, v, table, bucket_map, scale, key_mask, k_lens, cu_q, cu_k, max_q, max_k, causal, align_end,
                                        None if out is None else (out.shape, out.stride(), out.dtype), more)
    dev = q.device
    if not _rp_here(dev):
        with torch.cuda.device(dev):
            return relpos_attn_fwd(q, k, v, table, bucket_map, scale, key_mask, k_lens, cu_q, cu_k, max_q, max_k, causal, align_end, need_lse, out)
    if out is None:
        out = _rp_like(q)
    elif out.device != dev or out.data_ptr() & 15:
        raise ValueError(f"out must be on {dev}, its rows on 16 bytes")
    lse = table.new_empty(lse_shape, dtype=torch.float32) if need_lse else None
    ws = table.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    L.check(L.load().amdseg_relpos_attn_fwd(C.byref(c), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _p(lse), _p(ws), ws_bytes, _rp_s(dev)),
            "amdseg_relpos_attn_fwd")
    return out, lse


def relpos_attn_bwd(q, k, v, table, bucket_map, out, dout, lse, scale=None, key_mask=None, k_lens=None, cu_q=None, cu_k=None, max_q=None, max_k=None,
                    causal=False, align_end=False, need_dtable=True, dq=None, dk=None, dv=None):
    """gradients of relpos_attn_fwd from its `out` and `lse` (amdseg_relpos_attn_bwd): (dq, dk, dv, dtable), the last in the table's dtype or None.
    dq / dk / dv may be given (column blocks of one buffer): rows outside every packed sequence are left as they were in all three or, if none is given,
    zero.  Sums are taken in a fixed order: the same call gives the same bits."""
    if (dq is None) != (dk is None) or (dq is None) != (dv is None):
        raise ValueError("dq, dk, dv: give all three or none")

    def more(c, lse_shape):
        es = q.element_size()
        if out.shape != q.shape or dout.shape != q.shape or out.dtype != q.dtype or dout.dtype != q.dtype:
            raise ValueError(f"out and dout must be {tuple(q.shape)} {q.dtype}")
        if lse.shape != lse_shape or lse.dtype != torch.float32 or not lse.is_contiguous():
            raise ValueError(f"lse must be the contiguous fp32 {lse_shape} of relpos_attn_fwd")
        c.out_stride[:] = _rp_strides(out, "out", es)
        c.dout_stride[:] = _rp_strides(dout, "dout", es)
        c.zero_tail = int(dq is None)
        for name, t, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
            getattr(c, name + "_stride")[:] = _rp_dense(like.shape) if t is None else _rp_out(t, like, name, es)

    c, lse_shape, _, ws_bytes = _rp_cfg(q, k, v, table, bucket_map, scale, key_mask, k_lens, cu_q, cu_k, max_q, max_k, causal, align_end,
                                        (out.shape, out.stride(), out.dtype, dout.shape, dout.stride(), dout.dtype, lse.shape, lse.stride(), lse.dtype,
                                         dq is None or (dq.shape, dq.stride(), dq.dtype, dk.shape, dk.stride(), dk.dtype, dv.shape, dv.stride(), dv.dtype)), more)
    dev = q.device
    if not _rp_here(dev):
        with torch.cuda.device(dev):
            return relpos_attn_bwd(q, k, v, table, bucket_map, out, dout, lse, scale, key_mask, k_lens, cu_q, cu_k, max_q, max_k, causal, align_end, need_dtable,
                                   dq, dk, dv)
    if dq is None:
        dq, dk, dv = _rp_like(q), _rp_like(k), _rp_like(v)
    if out.device != dev or dout.device != dev or lse.device != dev or dq.device != dev or dk.device != dev or dv.device != dev:
        raise ValueError(f"out, dout, lse (and dq, dk, dv) must be on {dev}")
    at = out.data_ptr(), dout.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    if (at[0] | at[1] | at[3] | at[4] | at[5]) & 15:
        raise ValueError("out, dout (and dq, dk, dv): rows must start on 16 bytes")
    dtable = _rp_like(table) if need_dtable else None
    ws = table.new_empty(ws_bytes, dtype=torch.uint8)
    L.check(L.load().amdseg_relpos_attn_bwd(C.byref(c), q.data_ptr(), k.data_ptr(), v.data_ptr(), *at, _p(dtable), ws.data_ptr(), ws_bytes, _rp_s(dev)),
            "amdseg_relpos_attn_bwd")
    return dq, dk, dv, dtable


def relpos_bias_fwd(table, bucket_map, Lq, Lk, q_offset=0, out_dtype=torch.float32):
    """the bias of relpos_attn_fwd as a dense [heads, Lq, Lk] tensor: for attention composed from single operations (probabilities that are dropped out
    or returned)"""
    if table.dim() != 2 or Lq < 0 or Lk < 0:
        raise ValueError(f"table [buckets, heads], Lq and Lk >= 0, not {tuple(table.shape)}, {Lq}, {Lk}")
    c, dev, heads = L.RelposCfg(), table.device, table.shape[1]
    if dev.type == "cuda" and not _rp_here(dev):
        with torch.cuda.device(dev):
            return relpos_bias_fwd(table, bucket_map, Lq, Lk, q_offset, out_dtype)
    if dev.type != "cuda":
        raise ValueError("table must be on a GPU")
    _rp_table(c, table, bucket_map, heads)
    m = _rp_int(bucket_map, "bucket_map", bucket_map.numel(), dev)
    out = table.new_empty((heads, Lq, Lk), dtype=out_dtype)
    L.check(L.load().amdseg_relpos_bias_fwd(_p(table), c.table_dtype, m, c.span, c.buckets, heads, Lq, Lk, q_offset, _p(out), _dt(out), _rp_s(dev)),
            "amdseg_relpos_bias_fwd")
    return out


def relpos_bias_bwd(dbias, bucket_map, buckets, q_offset=0):
    """gradient of the table, fp32 [buckets, heads], from dbias [B, heads, Lq, Lk] (or [heads, Lq, Lk]), summed over the sequences, the queries and the
    distances of a bucket in a fixed order"""
    if dbias.dim() == 3:
        dbias = dbias.unsqueeze(0)
    if dbias.dim() != 4:
        raise ValueError(f"dbias must be [B, heads, Lq, Lk], not {tuple(dbias.shape)}")
    _chk(dbias, "dbias")
    B, heads, Lq, Lk = dbias.shape
    dev, n = dbias.device, bucket_map.numel()
    if n % 2 == 0 or n > 2049 or buckets < 1:
        raise ValueError(f"bucket_map must hold 2 * span + 1 entries with span <= 1024, not {n}; buckets = {buckets}")
    if dbias.data_ptr() & 15:
        raise ValueError("dbias must start on 16 bytes")
    m = _rp_int(bucket_map, "bucket_map", n, dev)
    if not _rp_here(dev):
        with torch.cuda.device(dev):
            return relpos_bias_bwd(dbias, bucket_map, buckets, q_offset)
    dtable = dbias.new_empty((buckets, heads), dtype=torch.float32)
    lib = L.load()
    ws_bytes = lib.amdseg_relpos_bias_ws_bytes(B, heads, Lq, n // 2)
    ws = dbias.new_empty(ws_bytes, dtype=torch.uint8)
    L.check(lib.amdseg_relpos_bias_bwd(_p(dbias), _dt(dbias), m, n // 2, buckets, B, heads, Lq, Lk, q_offset, _p(dtable), _p(ws), ws_bytes, _rp_s(dev)),
            "amdseg_relpos_bias_bwd")
    return dtable
