"""Attention with changed scores, as cases that can be timed: scores capped by a tanh or biased by distance, under window,
document and prefix masks.  Three operators: the packed form for training and prefill (``biased_attention``), its form for
one new token a sequence over a K/V cache (``biased_decode_attention``), and that form for batches whose sequences continue a
prefix that they share (``shared_prefix_decode_attention``).

    s = scale q.k;  s = cap tanh(s / cap);  s = s - slope_h |t - j|;  o = softmax(s over the visible j) v

Lists of lengths are texts ("300,212") so that a case is a dict of plain values.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
LOG2E = 1.4426950408889634


def _attn(name, train, seqlens, Hk, G, d, dtype, cap=0.0, alibi=False, window=0, docs="", prefix="", cached=""):
    """docs: lengths of the documents that the packed keys hold one after the other, negative for padding.  prefix: tokens at the
    start of every sequence that all of its tokens see.  cached: keys of every sequence in front of its queries."""
    return dict(name=name, kind="attn", train=train, seqlens=seqlens, Hk=Hk, G=G, d=d, dtype=dtype, cap=cap, alibi=alibi, window=window,
                docs=docs, prefix=prefix, cached=cached)


def _decode(name, lens, Hk, G, d, dtype, cap=0.0, alibi=False, window=0):
    return dict(name=name, kind="decode", lens=lens, Hk=Hk, G=G, d=d, dtype=dtype, cap=cap, alibi=alibi, window=window)


def _shared(name, prefixes, groups, lens, Hk, G, d, dtype, cap=0.0, alibi=False, window=0):
    """prefixes: lengths of the shared prefixes; groups: how many sequences continue each of them; lens: the sequences' own tokens."""
    return dict(name=name, kind="shared", prefixes=prefixes, groups=groups, lens=lens, Hk=Hk, G=G, d=d, dtype=dtype, cap=cap, alibi=alibi,
                window=window)


def listed():
    return [
        # a fine-tuning micro-batch or a test: two short packed sequences of a model with capped scores
        _attn("train_300_212_cap", True, "300,212", 2, 2, 128, "bf16", cap=50.0),
        # pretraining with distance biases on rows filled with documents, the ends of the rows padded
        _attn("train_2x4096_docs_alibi", True, "4096,4096", 8, 4, 128, "bf16", alibi=True,
              docs="1500,1,900,1300,-395,2777,640,65,300,-314"),
        # a long sequence in a local layer of a model with capped scores: the heads of the headline configuration
        _attn("train_16384_cap_window", True, "16384", 4, 2, 128, "bf16", cap=50.0, window=4096),
        # ... and in one of its global layers
        _attn("train_2x8192_cap", True, "8192,8192", 4, 2, 128, "bf16", cap=50.0),
        # narrow heads, ragged lengths, both changes of the score, fp16
        _attn("train_ragged_d64_fp16", True, "3001,777,2049,1365", 4, 4, 64, "fp16", cap=30.0, alibi=True),
        # one interactive prompt of a prefix model: its first part is read in both directions
        _attn("prefill_517_prefix", False, "517", 8, 4, 128, "bf16", cap=50.0, prefix="384"),
        # chunked prefill of long prompts: a chunk's queries against the cache and the chunk
        _attn("prefill_chunk_cap", False, "2048,333", 8, 4, 128, "bf16", cap=50.0, cached="17963,12012"),
        # one interactive request
        _decode("decode_1x8191_cap", "8191", 8, 4, 128, "bf16", cap=50.0),
        # a full batch with long caches of mixed lengths
        _decode("decode_64_ragged_alibi", ",".join(str(16384 - 193 * i) for i in range(64)), 8, 4, 128, "bf16", alibi=True),
        # a few requests that continue one system prompt
        _shared("shared_2048_x8_cap", "2048", "8", "1,77,300,15,512,128,9,64", 8, 4, 128, "bf16", cap=50.0),
        # a full batch that shares a long document
        _shared("shared_32768_x64", "32768", "64", ",".join(str(1 + (577 * i) % 1021) for i in range(64)), 8, 4, 128, "bf16", cap=50.0),
        # sampling many answers to three questions, narrow heads, distance biases
        _shared("shared_3_x200_d64_alibi", "9001,1,4100", "120,13,67", ",".join(str(1 + (97 * i) % 700) for i in range(200)), 4, 4, 64,
                "fp16", alibi=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _split(rng, total, parts):
    """``total`` in ``parts`` ragged pieces of at least one."""
    parts = min(parts, total)
    cuts = sorted(rng.sample(range(1, total), parts - 1)) if parts > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def _score(rng):
    """cap, alibi: at least one of them, mostly."""
    return rng.choice([(50.0, False), (30.0, False), (0.0, True), (50.0, True), (0.0, False)])


def draw(rng):
    kind = rng.choice(["attn", "attn", "decode", "shared"])
    d, dtype = rng.choice([128, 128, 64]), rng.choice(["bf16", "bf16", "fp16"])
    Hk, G = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8, 16])
    cap, alibi = _score(rng)
    if kind == "attn":
        train = rng.random() < 0.6
        while True:         # no more scores than the largest listed case has
            lens = _split(rng, _log_int(rng, 40, 16384), rng.choice([1, 1, 2, 4, 8]))
            form = rng.choice(["", "window", "docs", "prefix", "cached"])
            cached = [_log_int(rng, 1, 20000) if form == "cached" else 0 for _ in lens]
            if len(lens) * max(lens) * max(n + c for n, c in zip(lens, cached)) * Hk * G <= 10 ** 9:
                break
        docs = []
        if form == "docs":
            for n in lens:
                part = _split(rng, n, rng.choice([1, 2, 5, 9]))
                docs += part[:-1] + [-part[-1] if len(part) > 1 and rng.random() < 0.5 else part[-1]]
        c = _attn("", train, _text(lens), Hk, G, d, dtype, cap, alibi, window=_log_int(rng, 16, 4096) if form == "window" else 0,
                  docs=_text(docs), prefix=_text([rng.randrange(n + 1) for n in lens]) if form == "prefix" else "",
                  cached=_text(cached) if form == "cached" else "")
    elif kind == "decode":
        batch = _log_int(rng, 1, 64)
        longest = _log_int(rng, 40, 16384)
        lens = [longest] + [_log_int(rng, max(1, longest // 30), longest) for _ in range(batch - 1)]
        c = _decode("", _text(lens), Hk, G, d, dtype, cap, alibi, window=rng.choice([0, 0, _log_int(rng, 16, 4096)]))
    else:
        groups = [_log_int(rng, 1, 64) for _ in range(rng.choice([1, 1, 2, 3]))]
        prefixes = [_log_int(rng, 1, 32768 // len(groups)) for _ in groups]
        most = _log_int(rng, 1, 1024)
        c = _shared("", _text(prefixes), _text(groups), _text([_log_int(rng, 1, most) for _ in range(sum(groups))]), Hk, G, d, dtype, cap,
                    alibi, window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]))
    del c["name"]
    return c


def _ints(text):
    return [int(n) for n in text.split(",")] if text else []


def _cu(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


def _i32(numbers):
    return torch.tensor(numbers, dtype=torch.int32, device="cuda")


def _slopes(Hq):
    """The usual geometric sequence: 2^(-8 / Hq), 2^(-16 / Hq), ..."""
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / Hq) for i in range(Hq)], dtype=torch.float32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, Hk, d = DTYPES[case["dtype"]], case["Hk"], case["d"]
    Hq = Hk * case["G"]

    def rows(n, heads, size=1.0):
        return (torch.randn(n, heads, d, generator=g, device="cuda") * size).to(dt)

    s = dict(case=case, kind=case["kind"], scale=d ** -0.5, cap=case["cap"] or None, slopes=_slopes(Hq) if case["alibi"] else None,
             window=case["window"] or None)
    # queries of 3 standard deviations: scores reach 15 and more, as those of trained heads do
    if case["kind"] == "attn":
        lens = _ints(case["seqlens"])
        klens = [n + c for n, c in zip(lens, _ints(case["cached"]) or [0] * len(lens))]
        s.update(q=rows(sum(lens), Hq, 3.0), k=rows(sum(klens), Hk), v=rows(sum(klens), Hk), cu=_cu(lens), longest=max(lens),
                 longest_k=max(klens), train=case["train"], cu_k=_cu(klens) if case["cached"] else None,
                 prefix=_i32(_ints(case["prefix"])) if case["prefix"] else None, docs=None)
        if case["docs"]:
            ids = [torch.full((abs(n),), i if n > 0 else -1, dtype=torch.int32) for i, n in enumerate(_ints(case["docs"]))]
            s["docs"] = torch.cat(ids).cuda()
        if case["train"]:
            s["do"] = rows(sum(lens), Hq)
            for x in ("q", "k", "v"):
                s[x].requires_grad_()
        return s
    lens = _ints(case["lens"])
    cap = max(lens) + 1                         # a cache with a row to spare for every sequence
    s.update(q=rows(len(lens), Hq, 3.0), k=rows(len(lens) * cap, Hk), v=rows(len(lens) * cap, Hk), seq_len=_i32(lens),
             row0=_i32([cap * i for i in range(len(lens))]), max_len=max(lens))
    if case["kind"] == "shared":
        prefixes = _ints(case["prefixes"])
        s.update(pk=rows(sum(prefixes), Hk), pv=rows(sum(prefixes), Hk), cu_prefix=_cu(prefixes), cu_group=_cu(_ints(case["groups"])),
                 max_prefix=max(prefixes))
    return s


def run(s):
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "flash-sparse-attention_b200"))
        return _run_own(s)
    if s["kind"] == "decode":
        return _plain_decode(s)
    if s["kind"] == "shared":
        return _plain_shared(s)
    o, lse = _plain_attention(s)
    if not s["train"]:
        return o, lse
    return (o.detach(), lse.detach()) + torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])


def _run_own(s):
    how = dict(sm_scale=s["scale"], softcap=s["cap"], alibi_slopes=s["slopes"], window_size=s["window"])
    if s["kind"] == "decode":
        from fsa_preview.ops import biased_decode_attention

        return biased_decode_attention(s["q"], s["k"], s["v"], s["seq_len"], s["row0"], max_len=s["max_len"], **how)
    if s["kind"] == "shared":
        from fsa_preview.ops import shared_prefix_decode_attention

        return shared_prefix_decode_attention(s["q"], s["k"], s["v"], s["seq_len"], s["row0"], s["pk"], s["pv"], s["cu_prefix"], s["cu_group"],
                                              max_len=s["max_len"], max_prefix=s["max_prefix"], **how)
    from fsa.ops import biased_attention

    o, lse = biased_attention(s["q"], s["k"], s["v"], s["cu"], cu_seqlens_k=s["cu_k"], doc_ids=s["docs"], prefix_lens=s["prefix"], **how)
    if not s["train"]:
        return o, lse
    return (o.detach(), lse) + torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])


# ---------------------------------------------------------------------------------------------- plain forms, in 32 bits
def _change(x, s, slopes, dist):
    """Scores from products: cap and distance bias."""
    x = x * s["scale"]
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    return x if slopes is None else x - slopes * dist


def _softmax(x, seen):
    """exp(x - m), its sum and m over the seen keys of the last axis."""
    x = torch.where(seen, x, torch.full((), -math.inf, device=x.device))
    m = x.detach().amax(-1, keepdim=True)
    m = torch.where(m > -math.inf, m, torch.zeros_like(m))
    p = torch.exp(x - m)
    return p, p.sum(-1, keepdim=True), m


def _lse(l, m):
    return (m + torch.log(l)) * LOG2E


def _plain_attention(s):
    q, k, v, dev = s["q"], s["k"], s["v"], s["q"].device
    (N, Hq, d), (Nk, Hk) = q.shape, k.shape[:2]
    cu_k = s["cu"] if s["cu_k"] is None else s["cu_k"]
    B, Lq, Lk = s["cu"].numel() - 1, s["longest"], s["longest_k"]
    # every sequence into a row of its own
    tq, tk = torch.arange(N, device=dev), torch.arange(Nk, device=dev)
    bq, bk = (tq[:, None] >= s["cu"][None, 1:]).sum(1), (tk[:, None] >= cu_k[None, 1:]).sum(1)
    at_q, at_k = bq * Lq + tq - s["cu"][bq], bk * Lk + tk - cu_k[bk]
    qp = torch.zeros(B * Lq, Hq, d, device=dev).index_copy(0, at_q, q.float())
    kp = torch.zeros(B * Lk, Hk, d, device=dev).index_copy(0, at_k, k.float())
    vp = torch.zeros(B * Lk, Hk, d, device=dev).index_copy(0, at_k, v.float())
    qp = qp.view(B, Lq, Hk, Hq // Hk, d).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, d)       # [B, Hk, G Lq, d]
    kp, vp = kp.view(B, Lk, Hk, d).permute(0, 2, 1, 3), vp.view(B, Lk, Hk, d).permute(0, 2, 1, 3)
    # places in the sequence and who sees whom
    nq, nk = s["cu"].diff(), cu_k.diff()
    j = torch.arange(Lk, device=dev)
    t = torch.arange(Lq, device=dev)[None, :] + (nk - nq)[:, None]                          # [B, Lq]
    to = t if s["prefix"] is None else torch.maximum(t, s["prefix"][:, None] - 1)
    seen = (j <= to[..., None]) & (j < nk[:, None, None]) & (t < nk[:, None])[..., None]
    if s["window"]:
        seen &= j >= t[..., None] - s["window"]
    if s["docs"] is not None:
        of_k = torch.full((B * Lk,), -2, dtype=torch.int32, device=dev).index_copy(0, at_k, s["docs"]).view(B, Lk)
        of_q = torch.gather(of_k, 1, t.clamp(0, Lk - 1))
        seen &= (of_q[..., None] == of_k[:, None, :]) & (of_q >= 0)[..., None]
    slopes = None if s["slopes"] is None else s["slopes"].view(1, Hk, Hq // Hk, 1, 1)
    dist = (t[..., None] - j).abs().float()[:, None, None]                                  # [B, 1, 1, Lq, Lk]
    x = _change((qp @ kp.transpose(-1, -2)).view(B, Hk, -1, Lq, Lk), s, slopes, dist)
    p, l, m = _softmax(x, seen[:, None, None])
    o = (p.view(B, Hk, -1, Lk) @ vp).view(B, Hk, -1, Lq, d) / torch.where(l > 0, l, torch.ones_like(l))
    o = o.permute(0, 3, 1, 2, 4).reshape(B * Lq, Hq, d).index_select(0, at_q)
    lse = _lse(l.detach(), m)[..., 0].permute(0, 3, 1, 2).reshape(B * Lq, Hq).index_select(0, at_q)
    return o.to(q.dtype), lse.t().contiguous()


def _cache_part(s):
    """Unnormalised output, sum and maximum over every sequence's own rows of the cache, [B, Hk, G, ...]."""
    q, dev = s["q"], s["q"].device
    (B, Hq, d), Hk = q.shape, s["k"].shape[1]
    j = torch.arange(s["max_len"], device=dev)
    rows = (s["row0"][:, None] + j).clamp(max=s["k"].shape[0] - 1)
    kp, vp = s["k"][rows].float().permute(0, 2, 3, 1), s["v"][rows].float().permute(0, 2, 1, 3)     # [B, Hk, d, L], [B, Hk, L, d]
    t = s["seq_len"][:, None] - 1
    seen = j <= t
    if s["window"]:
        seen = seen & (j >= t - s["window"])
    slopes = None if s["slopes"] is None else s["slopes"].view(1, Hk, Hq // Hk, 1)
    x = _change(q.float().view(B, Hk, -1, d) @ kp, s, slopes, (t - j).float()[:, None, None])
    p, l, m = _softmax(x, seen[:, None, None])
    return p @ vp, l, m


def _plain_decode(s):
    o, l, m = _cache_part(s)
    o = (o / torch.where(l > 0, l, torch.ones_like(l))).to(s["q"].dtype)
    return o.flatten(1, 2), _lse(l, m)[..., 0].flatten(1, 2)


def _plain_shared(s):
    q, dev = s["q"], s["q"].device
    (B, Hq, d), (P, Hk) = q.shape, s["pk"].shape[:2]
    # all queries against all prefix rows at once: [Hk, G, B, P]
    x = q.float().view(B, Hk, -1, d).permute(1, 2, 0, 3).reshape(Hk, -1, d) @ s["pk"].float().permute(1, 2, 0)
    row, b = torch.arange(P, device=dev), torch.arange(B, device=dev)
    of_row, of_b = (row[:, None] >= s["cu_prefix"][None, 1:]).sum(1), (b[:, None] >= s["cu_group"][None, 1:]).sum(1)
    t = s["cu_prefix"].diff()[of_b] + s["seq_len"] - 1                                      # place of the new token
    j = row - s["cu_prefix"][of_row]
    seen = (of_row[None, :] == of_b[:, None]) & (s["seq_len"] > 0)[:, None]
    if s["window"]:
        seen &= j[None, :] >= t[:, None] - s["window"]
    slopes = None if s["slopes"] is None else s["slopes"].view(Hk, Hq // Hk, 1, 1)
    x = _change(x.view(Hk, -1, B, P), s, slopes, (t[:, None] - j).float())
    p, l, m = _softmax(x, seen)
    o = (p.view(Hk, -1, P) @ s["pv"].float().transpose(0, 1)).view(Hk, -1, B, d)
    o, l, m = (y.permute(2, 0, 1, 3) for y in (o, l, m))
    o2, l2, m2 = _cache_part(s)
    m = torch.where(l > 0, m, torch.full_like(m, -math.inf))
    m2 = torch.where(l2 > 0, m2, torch.full_like(m2, -math.inf))
    top = torch.maximum(m, m2)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    o, l = o * torch.exp(m - top) + o2 * torch.exp(m2 - top), l * torch.exp(m - top) + l2 * torch.exp(m2 - top)
    o = (o / torch.where(l > 0, l, torch.ones_like(l))).to(q.dtype)
    return o.flatten(1, 2), _lse(l, top)[..., 0].flatten(1, 2)


# ---------------------------------------------------------------------------------------------- what there is to do
def _pairs(case):
    """Visible (query, key) pairs of one head."""
    if case["kind"] == "attn":
        lens = _ints(case["seqlens"])
        cached, prefix, n = _ints(case["cached"]) or [0] * len(lens), _ints(case["prefix"]) or [0] * len(lens), 0
        if case["docs"]:
            return sum(x * (x + 1) // 2 for x in _ints(case["docs"]) if x > 0)
        for L, c, p in zip(lens, cached, prefix):
            w = case["window"] or L + c
            n += sum(min(max(t + 1, min(p, L)), w + 1) for t in range(c, c + L))
        return n
    lens = _ints(case["lens"])
    own_rows = [min(n, case["window"] + 1) if case["window"] else n for n in lens]
    if case["kind"] == "decode":
        return sum(own_rows)
    of = [i for i, n in enumerate(_ints(case["groups"])) for _ in range(n)]
    pre = _ints(case["prefixes"])
    return sum(own_rows) + sum(min(pre[g], max(0, case["window"] + 1 - n)) if case["window"] else pre[g] for g, n in zip(of, lens))


def work(case):
    Hk, d = case["Hk"], case["d"]
    Hq, pairs = Hk * case["G"], _pairs(case)
    if case["kind"] == "attn":
        N = sum(_ints(case["seqlens"]))
        Nk = N + sum(_ints(case["cached"]))
        io = 2 * d * (2 * N * Hq + 2 * Nk * Hk) + 4 * N * Hq                # q, o, k, v, lse
        if not case["train"]:
            return {"bytes": io, "flops": 4 * d * pairs * Hq}
        return {"bytes": io + 2 * d * (2 * N * Hq + 2 * Nk * Hk), "flops": 14 * d * pairs * Hq}       # dO, dq, dk, dv
    lens = _ints(case["lens"])
    rows = sum(min(n, case["window"] + 1) if case["window"] else n for n in lens)
    if case["kind"] == "shared":
        first, pre = 0, _ints(case["prefixes"])
        for g, n in enumerate(_ints(case["groups"])):
            near = min(lens[first : first + n])                             # the sequence that looks furthest back
            rows += min(pre[g], max(0, case["window"] + 1 - near)) if case["window"] else pre[g]
            first += n
    return {"bytes": 2 * d * (2 * rows * Hk + 2 * len(lens) * Hq) + 4 * len(lens) * Hq, "flops": 4 * d * pairs * Hq}


# ---------------------------------------------------------------------------------------------- in 64 bits, head by head
def _exact_rows(q, k, v, seen, dist, cap, slope, scale, do=None):
    """One head of one sequence: o, lse [, dq, dk, dv]."""
    x = scale * (q @ k.T)
    th = torch.tanh(x / cap) if cap else None
    x = cap * th if cap else x
    x = x - slope * dist if slope else x
    x = x.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(x, 1, keepdim=True)
    p = torch.exp(x - lse).masked_fill(~seen, 0.0)
    o = p @ v
    if do is None:
        return o, lse[:, 0] / math.log(2.0)
    ds = p * (do @ v.T - (o * do).sum(1, keepdim=True)) * scale
    ds = ds * (1 - th * th) if cap else ds
    return o, lse[:, 0] / math.log(2.0), ds @ k, ds.T @ q, p.T @ do


def exact(case, seed):
    s = prepare(case, seed)
    Hk, G = case["Hk"], case["G"]
    q, k, v = (s[x].detach().double() for x in "qkv")
    cap, slopes = case["cap"], s["slopes"].tolist() if case["alibi"] else [0.0] * (Hk * G)
    o, lse = torch.zeros_like(q), torch.full((Hk * G, q.shape[0]), -math.inf, dtype=torch.float64, device="cuda")
    if case["kind"] == "attn":
        do = s["do"].double() if case["train"] else None
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        lens = _ints(case["seqlens"])
        cached, prefix = _ints(case["cached"]) or [0] * len(lens), _ints(case["prefix"]) or [0] * len(lens)
        a = b = 0
        for L, c, pre in zip(lens, cached, prefix):
            qs, ks = slice(a, a + L), slice(b, b + L + c)
            a, b = a + L, b + L + c
            t, j = torch.arange(c, c + L, device="cuda")[:, None], torch.arange(L + c, device="cuda")[None, :]
            seen = (j <= t) | (j < pre)
            if case["window"]:
                seen = seen & (t - j <= case["window"])
            if s["docs"] is not None:
                ids = s["docs"][ks]
                seen = seen & (ids[c:, None] == ids[None, :]) & (ids[c:, None] >= 0)
            for h in range(Hk * G):
                kv = h // G
                got = _exact_rows(q[qs, h], k[ks, kv], v[ks, kv], seen, (t - j).abs(), cap, slopes[h], s["scale"], do[qs, h] if case["train"] else None)
                o[qs, h], lse[h, qs] = got[:2]
                if case["train"]:
                    dq[qs, h] = got[2]
                    dk[ks, kv] += got[3]
                    dv[ks, kv] += got[4]
        return (o, lse, dq, dk, dv) if case["train"] else (o, lse)
    lens = _ints(case["lens"])
    of = [i for i, n in enumerate(_ints(case.get("groups", ""))) for _ in range(n)]
    starts = [0]
    for n in _ints(case.get("prefixes", "")):
        starts.append(starts[-1] + n)
    for b, n in enumerate(lens):
        r0 = b * (max(lens) + 1)
        kb, vb = k[r0 : r0 + n], v[r0 : r0 + n]
        if of:
            pre = slice(starts[of[b]], starts[of[b] + 1])
            kb, vb = torch.cat([s["pk"][pre].double(), kb]), torch.cat([s["pv"][pre].double(), vb])
        back = torch.arange(kb.shape[0] - 1, -1, -1, device="cuda")[None, :]
        seen = back <= case["window"] if case["window"] else back >= 0
        for h in range(Hk * G):
            got = _exact_rows(q[b : b + 1, h], kb[:, h // G], vb[:, h // G], seen, back, cap, slopes[h], s["scale"])
            o[b, h], lse[h, b] = got[0][0], got[1][0]
    return o, lse.t()
