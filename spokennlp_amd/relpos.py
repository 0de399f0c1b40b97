"""Attention under a learned relative position bias, as differentiable functions and a layer's module over the kernels of ``ops.relpos_*``.

The reference's encoders add learned ABSOLUTE position embeddings to the tokens ([hf] models/bert/modeling_bert.py:53-108); encoders that instead learn one
scalar per (bucket of distance, head) and add it to the attention scores run here on the same layers' projections:

    s_ij = scale q_i . k_j + table[bucket(j - i), head],   out_i = sum_j softmax_j(s_ij) v_j

Sequences come padded with a key mask, packed without padding (``cu_seqlens``), or as a cache with its fill (``k_lens``); see ``ops.relpos_attn_fwd``.
bf16 or fp32; there is no dropout on the probabilities (compose ``relpos_bias`` with single operations where it is needed)."""
import math

import torch
import torch.nn as nn

from . import ops


def _rows_ok(t):
    """whether the kernels take t's strides as they are"""
    es = t.element_size()
    return t.stride(-1) == 1 and all(s * es % 16 == 0 and s * es <= 1 << 24 for s, n in zip(t.stride()[-3:-1], t.shape[-3:-1]) if n > 1) and \
        (t.dim() < 4 or t.shape[0] == 1 or t.stride(0) * es % 16 == 0) and t.data_ptr() % 16 == 0


def _rows(t):
    """t as the kernels take it: a gradient may come with any strides, or contiguous from any element of a larger one (then contiguous() is t itself)"""
    if _rows_ok(t):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _RelposAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, bucket_map, how):
        out, lse = ops.relpos_attn_fwd(q, k, v, table, bucket_map, need_lse=any(ctx.needs_input_grad[:4]), **how)
        ctx.save_for_backward(q, k, v, table, bucket_map, out, lse, *(how[n] for n in ("key_mask", "k_lens", "cu_q", "cu_k")))
        ctx.how = {n: x for n, x in how.items() if n not in ("key_mask", "k_lens", "cu_q", "cu_k")}
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, table, bucket_map, out, lse, key_mask, k_lens, cu_q, cu_k = ctx.saved_tensors
        dq, dk, dv, dtable = ops.relpos_attn_bwd(q, k, v, table, bucket_map, out, _rows(dout), lse, need_dtable=ctx.needs_input_grad[3], key_mask=key_mask,
                                                 k_lens=k_lens, cu_q=cu_q, cu_k=cu_k, **ctx.how)
        return dq, dk, dv, dtable, None, None


class _RelposSelfAttention(torch.autograd.Function):
    """the same on the column blocks of one fused projection; the gradient is written as the fused tensor too"""

    @staticmethod
    def _blocks(t, heads, kv_heads):
        D = t.shape[-1] // (heads + 2 * kv_heads)
        return [x.unflatten(-1, (-1, D)) for x in t.split([heads * D, kv_heads * D, kv_heads * D], -1)]

    @staticmethod
    def forward(ctx, qkv, table, bucket_map, heads, kv_heads, how):
        q, k, v = _RelposSelfAttention._blocks(qkv, heads, kv_heads)
        out, lse = ops.relpos_attn_fwd(q, k, v, table, bucket_map, need_lse=any(ctx.needs_input_grad[:2]), **how)
        ctx.save_for_backward(qkv, table, bucket_map, out, lse, *(how[n] for n in ("key_mask", "cu_q", "cu_k")))
        ctx.how = {n: x for n, x in how.items() if n not in ("key_mask", "cu_q", "cu_k")}
        ctx.heads = (heads, kv_heads)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        qkv, table, bucket_map, out, lse, key_mask, cu_q, cu_k = ctx.saved_tensors
        q, k, v = _RelposSelfAttention._blocks(qkv, *ctx.heads)
        # packed: the rows outside every sequence are left alone by the kernels, and their gradient is zero
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device) if cu_q is None else torch.zeros(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        dq, dk, dv = _RelposSelfAttention._blocks(dqkv, *ctx.heads)
        dtable = ops.relpos_attn_bwd(q, k, v, table, bucket_map, out, _rows(dout), lse, need_dtable=ctx.needs_input_grad[1], key_mask=key_mask, cu_q=cu_q, cu_k=cu_k,
                                     dq=dq, dk=dk, dv=dv, **ctx.how)[3]
        return dqkv, dtable, None, None, None, None


class _RelposBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, bucket_map, Lq, Lk, q_offset, out_dtype):
        ctx.save_for_backward(bucket_map)
        ctx.of = (table.shape[0], table.dtype, q_offset)
        return ops.relpos_bias_fwd(table, bucket_map, Lq, Lk, q_offset, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dbias):
        buckets, dtype, q_offset = ctx.of
        dbias = dbias.contiguous()
        if dbias.data_ptr() % 16:                            # (a contiguous slice of a larger gradient)
            dbias = dbias.clone()
        return ops.relpos_bias_bwd(dbias, ctx.saved_tensors[0], buckets, q_offset).to(dtype), None, None, None, None, None


def relpos_attention(q, k, v, table, bucket_map, *, scale=None, key_mask=None, k_lens=None, cu_q=None, cu_k=None, max_q=None, max_k=None, causal=False,
                     align_end=False):
    """differentiable ops.relpos_attn_fwd: out with q's shape; gradients for q, k, v and the table"""
    how = dict(scale=None if scale is None else float(scale), key_mask=key_mask, k_lens=k_lens, cu_q=cu_q, cu_k=cu_k, max_q=max_q, max_k=max_k, causal=causal, align_end=align_end)
    return _RelposAttention.apply(q, k, v, table, bucket_map, how)


def relpos_self_attention(qkv, heads, table, bucket_map, *, kv_heads=None, scale=None, key_mask=None, cu_seqlens=None, longest=None, causal=False):
    """self-attention on a fused projection [B, L, (heads + 2 kv_heads) D] (packed: [tokens, ...] with cu_seqlens int32 [B + 1]): out [..., heads * D].  No copy
    of q, k or v is made, the gradient of the projection is one tensor."""
    kv_heads = kv_heads or heads
    if qkv.shape[-1] % (heads + 2 * kv_heads):
        raise ValueError(f"a projection of {qkv.shape[-1]} columns does not hold {heads} + 2 * {kv_heads} heads")
    how = dict(scale=None if scale is None else float(scale), key_mask=key_mask, cu_q=cu_seqlens, cu_k=cu_seqlens, max_q=longest, max_k=longest, causal=causal)
    return _RelposSelfAttention.apply(qkv, table, bucket_map, heads, kv_heads, how).flatten(-2)


def relpos_bias(table, bucket_map, Lq, Lk, q_offset=0, out_dtype=torch.float32):
    """differentiable ops.relpos_bias_fwd: the dense bias [heads, Lq, Lk]"""
    return _RelposBias.apply(table, bucket_map, Lq, Lk, q_offset, out_dtype)


class RelPosSelfAttention(nn.Module):
    """a layer's self-attention with bucketed relative positions: fused projection, attention, output projection.  ``table`` [buckets, heads] is the module's own
    unless one is given (layers that share their positions pass the first layer's)."""

    def __init__(self, hidden_size, heads, kv_heads=None, buckets=32, max_distance=128, bidirectional=True, bias=True, table=None):
        super().__init__()
        kv_heads = kv_heads or heads
        if hidden_size % heads or heads % kv_heads:
            raise ValueError(f"hidden size {hidden_size}, {heads} heads, {kv_heads} key / value heads")
        self.heads, self.kv_heads, self.bidirectional = heads, kv_heads, bidirectional
        D = hidden_size // heads
        self.qkv = nn.Linear(hidden_size, (heads + 2 * kv_heads) * D, bias=bias)
        self.out = nn.Linear(hidden_size, hidden_size, bias=bias)
        if table is None:
            table = nn.Parameter(torch.empty(buckets, heads).normal_(std=1.0 / math.sqrt(hidden_size)))
        elif tuple(table.shape) != (buckets, heads):
            raise ValueError(f"table must be [{buckets}, {heads}], not {tuple(table.shape)}")
        self.table = table
        self.register_buffer("bucket_map", torch.tensor(ops.relpos_bucket_list(buckets, max_distance, bidirectional), dtype=torch.int32), persistent=False)

    def forward(self, x, key_mask=None, cu_seqlens=None, longest=None):
        """x [B, L, H] with key_mask [B, L], or packed [tokens, H] with cu_seqlens"""
        ctx = relpos_self_attention(self.qkv(x), self.heads, self.table, self.bucket_map, kv_heads=self.kv_heads, key_mask=key_mask, cu_seqlens=cu_seqlens,
                                    longest=longest, causal=not self.bidirectional)
        return self.out(ctx)
