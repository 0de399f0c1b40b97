"""The relative-position attention operators as cases that can be timed: forward, forward + backward, and the dense bias with its gradient.

Every case says whether it is one self-attention batch of padded windows, a packed batch of ragged sequences, or a few queries against a
cache.  ``own`` selects who computes: False = elementary torch operations in fp32 on the same inputs, True = the calls a user makes of
``spokennlp_amd.ops``.
"""
import math
import random

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _case(name, op, dtype, form, B, Lq, Lk, heads, kv_heads, D, **more):
    c = dict(name=name, op=op, dtype=dtype, form=form, B=B, Lq=Lq, Lk=Lk, heads=heads, kv_heads=kv_heads, D=D, buckets=32, max_distance=128,
             causal=False, shortest=Lk, masked=False, tail=0, lseed=1)
    c.update(more)
    return c


def listed():
    return [
        # the fine-tuning step's layer: 32 windows of 512 tokens, 12 heads of 64, the windows of document ends padded
        _case("train_32x512", "train", "bf16", "padded", 32, 512, 512, 12, 12, 64, shortest=60, masked=True),
        # long documents in one window
        _case("train_4x4096", "train", "bf16", "padded", 4, 4096, 4096, 12, 12, 64, shortest=2500, masked=True),
        # the same work without padding: sequences of very different lengths behind one another, some buffer rows unused
        _case("train_packed", "train", "bf16", "packed", 24, 1500, 1500, 12, 12, 64, shortest=1, tail=37, lseed=5),
        # a wider model whose query heads share key / value heads, one-sided positions, odd length
        _case("train_shared_causal", "train", "bf16", "padded", 3, 1023, 1023, 16, 4, 128, causal=True),
        # reference precision
        _case("train_fp32", "train", "fp32", "padded", 4, 384, 384, 12, 12, 64, shortest=200, masked=True),
        # a few short sentences: latency
        _case("train_small", "train", "bf16", "padded", 2, 33, 33, 4, 4, 32),
        # inference over a batch of windows
        _case("infer_32x512", "infer", "bf16", "padded", 32, 512, 512, 12, 12, 64, shortest=60, masked=True),
        # one whole meeting transcript
        _case("infer_1x16384", "infer", "bf16", "padded", 1, 16384, 16384, 12, 12, 64),
        # one sentence: latency
        _case("infer_small", "infer", "bf16", "padded", 1, 64, 64, 12, 12, 64),
        # single tokens against caches of unlike fill
        _case("infer_token", "infer", "bf16", "cache", 16, 1, 4096, 16, 4, 128, causal=True, shortest=700),
        # dense bias for attention composed from single operations (dropout on the probabilities), and its gradient
        _case("bias_512", "bias", "bf16", "padded", 8, 512, 512, 12, 12, 64),
        _case("bias_odd", "bias", "fp32", "padded", 2, 1537, 2049, 12, 12, 64, buckets=64, max_distance=200),
    ]


def draw(rng):
    def log(a, b):
        return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b + 0.49)))))))

    while True:
        op = rng.choice(("train", "train", "infer", "infer", "bias"))
        form = "padded" if op == "bias" else rng.choice(("padded", "packed", "cache") if op == "infer" else ("padded", "padded", "packed"))
        kv = rng.choice((1, 2, 4, 6, 8, 12))
        heads = kv * rng.choice((1, 1, 2, 4))
        D = rng.choice((16, 32, 40, 64, 64, 80, 96, 128))
        dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
        B = log(1, 32)
        Lk = log(1, 8192)
        Lq = Lk
        if form == "cache":
            Lq = min(Lk, log(1, 64))
        elif op == "bias" or (form == "padded" and rng.random() < 0.25):
            Lq = log(1, 4096)
        two = rng.random() < 0.7
        c = _case("", op, dtype, form, B, Lq, Lk, heads, kv, D, buckets=rng.choice((8, 32, 32, 64)), max_distance=rng.choice((48, 128, 128, 200, 512)),
                  causal=op != "bias" and not two and (form != "padded" or Lq == Lk),
                  masked=form == "padded" and op != "bias" and rng.random() < 0.6, tail=rng.choice((0, 0, 5, 64)) if form == "packed" else 0,
                  lseed=rng.randrange(1, 10 ** 6))
        c["shortest"] = rng.randint(1, Lk) if (c["masked"] or form != "padded") else Lk
        del c["name"]
        pairs = B * heads * Lq * Lk
        if op == "bias":
            if 10 ** 4 <= pairs <= 8e7:
                return c
        elif 10 ** 4 <= pairs and pairs * D * (14 if op == "train" else 4) * (6 if dtype == "fp32" else 1) <= 7e11 and pairs <= 8e8:
            return c


# ------------------------------------------------------------------------------------------------ inputs
def _lens(case):
    """visible keys (and, packed, tokens) of every sequence: the first one is full, the rest spread down to the shortest"""
    r = random.Random(case["lseed"])
    return [case["Lk"]] + [r.randint(case["shortest"], case["Lk"]) for _ in range(case["B"] - 1)]


def _cum(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _two_sided(case):
    return not case["causal"]


def _bucket_list(case):
    """bucket of rel = -max_distance .. max_distance: small distances each their own, larger ones by steps that grow like the distance, two
    halves for the two signs unless one-sided.  Whole-number comparisons: n >= m (M / m)^(k / steps)  <=>  n^steps >= m^(steps - k) M^k"""
    nb, M = case["buckets"], case["max_distance"]
    half = nb // 2 if _two_sided(case) else nb
    m = half // 2
    steps = half - m

    def near(n):
        if n < m:
            return n
        k = 0
        while k + 1 < steps and n ** steps >= m ** (steps - k - 1) * M ** (k + 1):
            k += 1
        return m + k

    out = []
    for rel in range(-M, M + 1):
        if _two_sided(case):
            out.append(near(abs(rel)) + (half if rel > 0 else 0))
        else:
            out.append(near(max(-rel, 0)))
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed % 2 ** 31) + 17)
    dt, D, Hq, Hk = DTYPE[case["dtype"]], case["D"], case["heads"], case["kv_heads"]

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    s = {"case": case, "map": torch.tensor(_bucket_list(case), dtype=torch.int32, device="cuda")}
    B, Lq, Lk = case["B"], case["Lq"], case["Lk"]
    if case["op"] == "bias":
        s["table"] = randn(case["buckets"], Hq, dtype=torch.float32)
        s["dbias"] = randn(B, Hq, Lq, Lk)
        return s
    s["table"] = randn(case["buckets"], Hq)
    lens = _lens(case)
    if case["form"] == "packed":
        cu = _cum(lens)
        T = cu[-1] + case["tail"]
        lead_q, lead_k = (T,), (T,)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        s["longest"] = max(lens)
    else:
        lead_q, lead_k = (B, Lq), (B, Lk)
    if case["form"] == "cache" or Lq != Lk:
        s["q"], s["k"], s["v"] = randn(*lead_q, Hq, D), randn(*lead_k, Hk, D), randn(*lead_k, Hk, D)
    else:                                                    # column blocks of one fused projection, as a layer has them
        qkv = randn(*lead_q, (Hq + 2 * Hk) * D)
        s["q"] = qkv[..., :Hq * D].unflatten(-1, (Hq, D))
        s["k"] = qkv[..., Hq * D:(Hq + Hk) * D].unflatten(-1, (Hk, D))
        s["v"] = qkv[..., (Hq + Hk) * D:].unflatten(-1, (Hk, D))
    if case["masked"]:
        s["key_mask"] = torch.arange(Lk, device="cuda")[None, :] < torch.tensor(lens, device="cuda")[:, None]
    if case["form"] == "cache":
        s["k_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if case["op"] == "train":
        s["dout"] = randn(*lead_q, Hq, D)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def _own(s):
    from spokennlp_amd import ops
    c = s["case"]
    if c["op"] == "bias":
        bias = ops.relpos_bias_fwd(s["table"], s["map"], c["Lq"], c["Lk"], out_dtype=DTYPE[c["dtype"]])
        return {"bias": bias, "dtable": ops.relpos_bias_bwd(s["dbias"], s["map"], c["buckets"])}
    how = dict(causal=c["causal"])
    if c["form"] == "packed":
        how.update(cu_q=s["cu"], cu_k=s["cu"], max_q=s["longest"], max_k=s["longest"])
    if c["form"] == "cache":
        how.update(k_lens=s["k_lens"], align_end=True)
    if "key_mask" in s:
        how.update(key_mask=s["key_mask"])
    if c["op"] == "infer":
        return {"out": ops.relpos_attn_fwd(s["q"], s["k"], s["v"], s["table"], s["map"], need_lse=False, **how)[0]}
    out, lse = ops.relpos_attn_fwd(s["q"], s["k"], s["v"], s["table"], s["map"], **how)
    dq, dk, dv, dtable = ops.relpos_attn_bwd(s["q"], s["k"], s["v"], s["table"], s["map"], out, s["dout"], lse, **how)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}


def _rel_index(s, Lq, Lk, off):
    """[.., Lq, Lk] position in the map of every (query, key), and rel itself; off: None or [B] added to the query's position"""
    span = s["map"].numel() // 2
    rel = torch.arange(Lk, device="cuda")[None, :] - torch.arange(Lq, device="cuda")[:, None]
    if off is not None:
        rel = rel[None] - off[:, None, None]
    return rel.clamp(-span, span) + span, rel


def _table_gradient(s, d):
    """d [heads, Lq, Lk] in 64 bits -> [buckets, heads]: first the sums over the places of equal rel (rows turned over and re-cut one element
    shorter, so that equal rel share a column), then over the distances of a bucket"""
    H, Lq, Lk = d.shape
    wide = torch.cat((d.flip(1), d.new_zeros(H, Lq, Lq)), 2).flatten(1)[:, :Lq * (Lq + Lk - 1)]
    by_rel = wide.view(H, Lq, Lq + Lk - 1).sum(1)                                   # column n: rel = n - (Lq - 1)
    span = s["map"].numel() // 2
    bucket = s["map"].long()[torch.arange(1 - Lq, Lk, device="cuda").clamp(-span, span) + span]
    hot = (bucket[:, None] == torch.arange(s["case"]["buckets"], device="cuda")[None, :]).double()
    return torch.matmul(by_rel, hot).t().contiguous()


def _plain_bias(s):
    c = s["case"]
    dt = DTYPE[c["dtype"]]
    at, _ = _rel_index(s, c["Lq"], c["Lk"], None)
    bucket = s["map"].long()[at]
    bias = s["table"].float()[bucket].permute(2, 0, 1).to(dt).contiguous()
    return {"bias": bias, "dtable": _table_gradient(s, s["dbias"].sum(0, dtype=torch.float64)).float()}


def _to_padded(x, cu, longest):
    """[T, ...] -> [B, longest, ...], rows past a sequence's end zero; and the padded places that hold a token"""
    B = cu.numel() - 1
    at = cu[:-1, None].long() + torch.arange(longest, device="cuda")[None, :]
    held = at < cu[1:, None]
    got = x[torch.where(held, at, torch.zeros_like(at))]
    return got * held.view(B, longest, *([1] * (x.dim() - 1))), held


def _to_packed(x, held, T):
    """the inverse; the buffer's rows behind the last sequence are zero"""
    n = held.flatten().cumsum(0) - 1
    at = torch.where(held.flatten(), n, torch.full_like(n, T))                      # places without a token go to a row that is cut off
    wide = torch.zeros(T + 1, *x.shape[2:], dtype=x.dtype, device="cuda")
    wide[at] = x.flatten(0, 1)
    return wide[:T]


def _plain(s):
    c = s["case"]
    if c["op"] == "bias":
        return _plain_bias(s)
    dt, Hq, Hk, D = DTYPE[c["dtype"]], c["heads"], c["kv_heads"], c["D"]
    G, scale = Hq // Hk, D ** -0.5
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    dout = s["dout"].float() if "dout" in s else None
    held, off = None, None
    if c["form"] == "packed":
        T = q.shape[0]
        q, held = _to_padded(q, s["cu"], s["longest"])
        k, _ = _to_padded(k, s["cu"], s["longest"])
        v, _ = _to_padded(v, s["cu"], s["longest"])
        if dout is not None:
            dout, _ = _to_padded(dout, s["cu"], s["longest"])
    B, Lq, Lk = q.shape[0], q.shape[1], k.shape[1]
    if c["form"] == "cache":
        off = s["k_lens"].long() - Lq
    at, rel = _rel_index(s, Lq, Lk, off)
    bucket = s["map"].long()[at]                                                    # [Lq, Lk] or [B, Lq, Lk]
    bias = s["table"].float()[bucket].movedim(-1, -3).unflatten(-3, (Hk, G))        # [(B,) Hk, G, Lq, Lk]
    seen = None
    if held is not None:
        seen = held[:, None, None, None, :]
    if "key_mask" in s:
        seen = s["key_mask"][:, None, None, None, :]
    if "k_lens" in s:
        seen = (torch.arange(Lk, device="cuda")[None, :] < s["k_lens"][:, None])[:, None, None, None, :]
    if c["causal"]:
        past = (rel <= 0) if rel.dim() == 2 else (rel <= 0)[:, None, None]
        seen = past if seen is None else seen & past
    qh = q.permute(0, 2, 1, 3).unflatten(1, (Hk, G))                                # [B, Hk, G, Lq, D]
    kh, vh = k.permute(0, 2, 1, 3)[:, :, None], v.permute(0, 2, 1, 3)[:, :, None]   # [B, Hk, 1, Lk, D]
    p = torch.matmul(qh, kh.transpose(-1, -2)) * scale + bias
    if seen is not None:
        p = p.masked_fill(~seen, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    oh = torch.matmul(p, vh)

    def back(x, n):                                                                 # [B, n, L, D] -> the caller's layout
        x = x.permute(0, 2, 1, 3)
        if held is not None:
            x = _to_packed(x, held, T)
        return x.to(dt).contiguous()

    out = back(oh.flatten(1, 2), Hq)
    if dout is None:
        return {"out": out}
    doh = dout.permute(0, 2, 1, 3).unflatten(1, (Hk, G))
    dvh = torch.matmul(p.transpose(-1, -2), doh).sum(2)
    ds = torch.matmul(doh, vh.transpose(-1, -2))
    ds = p * (ds - (ds * p).sum(-1, keepdim=True))
    del p
    dqh = torch.matmul(ds, kh) * scale
    dkh = torch.matmul(ds.transpose(-1, -2), qh).sum(2) * scale
    dtable = _table_gradient(s, ds.sum(0, dtype=torch.float64).flatten(0, 1)).to(dt)
    return {"out": out, "dq": back(dqh.flatten(1, 2), Hq), "dk": back(dkh, Hk), "dv": back(dvh, Hk), "dtable": dtable}


def run(state):
    with torch.no_grad():
        if own:
            return _own(state)
        return _plain(state)


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    Hq, Hk, D, B, Lq, Lk = case["heads"], case["kv_heads"], case["D"], case["B"], case["Lq"], case["Lk"]
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "bias":
        return {"bytes": float(e * Hq * Lq * Lk * (1 + B)), "flops": float(B * Hq * Lq * Lk)}
    lens = _lens(case)
    if case["form"] == "packed":
        nq, pairs = sum(lens), sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        nk = nq
    else:
        nq, nk, pairs = B * Lq, sum(lens), 0
        for n in lens:
            if not case["causal"]:
                pairs += Lq * n
            else:                                                                   # query i sees keys 0 .. i + off
                off = n - Lq if case["form"] == "cache" else 0
                pairs += sum(max(0, min(n, i + off + 1)) for i in range(Lq))
    train = case["op"] == "train"
    rows = nq * Hq * D * (4 if train else 2) + nk * Hk * D * (4 if train else 2)
    return {"bytes": float(rows * e), "flops": float((14 if train else 4) * D * Hq * pairs)}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    lut = torch.tensor(_bucket_list(case), device="cuda")
    M = case["max_distance"]
    Hq, Hk, D = case["heads"], case["kv_heads"], case["D"]
    G = Hq // Hk
    if case["op"] == "bias":
        Lq, Lk = case["Lq"], case["Lk"]
        i, j = torch.arange(Lq, device="cuda").view(-1, 1), torch.arange(Lk, device="cuda").view(1, -1)
        which = lut[(torch.clamp(j - i, min=-M, max=M) + M)]
        table = s["table"].to(f64)
        bias = torch.stack([table[:, h][which] for h in range(Hq)])
        hot = [(which == n) for n in range(case["buckets"])]
        d = s["dbias"].to(f64).sum(0)
        dtable = torch.stack([torch.stack([d[h][m].sum() for h in range(Hq)]) for m in hot])
        return {"bias": bias, "dtable": dtable}
    train = case["op"] == "train"
    lens = _lens(case)
    cu = _cum(lens)
    table = s["table"].to(f64).requires_grad_(train)
    out = torch.zeros(s["q"].shape, dtype=f64, device="cuda")
    dq, dk, dv = torch.zeros_like(out), torch.zeros(s["k"].shape, dtype=f64, device="cuda"), torch.zeros(s["k"].shape, dtype=f64, device="cuda")
    dtable = torch.zeros_like(table.detach())
    for b in range(case["B"]):
        if case["form"] == "packed":
            at_q = at_k = (slice(cu[b], cu[b + 1]),)
        else:
            at_q, at_k = (b, slice(None)), (b, slice(0, lens[b]))
        first = lens[b] - case["Lq"] if case["form"] == "cache" else 0
        nq = s["q"][at_q].shape[0]
        rel = torch.arange(lens[b], device="cuda").view(1, -1) - (torch.arange(nq, device="cuda").view(-1, 1) + first)
        which = lut[torch.clamp(rel, min=-M, max=M) + M]
        for h in range(Hq):
            q = s["q"][at_q + (h,)].to(f64).requires_grad_(train)
            k = s["k"][at_k + (h // G,)].to(f64).requires_grad_(train)
            v = s["v"][at_k + (h // G,)].to(f64).requires_grad_(train)
            col = table[:, h]
            score = (q @ k.t()) / math.sqrt(D) + col[which]
            if case["causal"]:
                score = torch.where(rel > 0, torch.full_like(score, -math.inf), score)
            blind = (score == -math.inf).all(1)
            p = torch.softmax(torch.where(blind[:, None], torch.zeros_like(score), score), 1) * (~blind)[:, None]
            o = p @ v
            out[at_q + (h,)] = o.detach()
            if train:
                gq, gk, gv, gt = torch.autograd.grad(o, (q, k, v, table), s["dout"][at_q + (h,)].to(f64))
                dq[at_q + (h,)] = gq
                dk[at_k + (h // G,)] += gk
                dv[at_k + (h // G,)] += gv
                dtable += gt
    if not train:
        return {"out": out}
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}
