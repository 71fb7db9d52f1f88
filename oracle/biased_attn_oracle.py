"""Attention with changed scores and masks from its definition, in 64 bits on the CPU, with what its roundings may add up to.

    s = scale q.k;  s = cap tanh(s / cap);  s = s - slope_h |t - j|;  o = softmax(s over the visible j) v

Every function works on one packed batch, sequence by sequence and head by head.
"""
from __future__ import annotations

import math

import torch


def visible(Lq, Lk, window=None, ids=None, prefix=None):
    """[Lq, Lk] who sees whom, and |t - j|; the queries are the last Lq of the Lk places (they may begin before the first)."""
    t = torch.arange(Lk - Lq, Lk)[:, None]
    j = torch.arange(Lk)[None, :]
    seen = j <= t
    if prefix is not None:
        seen = seen | ((j < prefix) & (t >= 0))
    if window is not None:
        seen = seen & (j >= t - window)
    if ids is not None and Lk:
        # stretches of equal ids
        run = torch.cumsum(torch.cat([torch.zeros(1, dtype=torch.long), (ids[1:] != ids[:-1]).long()]), 0)
        at = t[:, 0].clamp(min=0)
        seen = seen & (run[at][:, None] == run[None, :]) & (ids[at] >= 0)[:, None]
    return seen, (t - j).abs().double()


def one_head(q, k, v, seen, dist, scale, cap=0.0, slope=0.0, do=None, half=0.0, tiny=0.0):
    """o, lse (log2 units), and with ``do`` also dq, dk, dv; then for each of o, dq, dk, dv the most that roundings to the 16-bit type can
    make of it: ``half`` of a step relative to each of P, dS, o and the results, ``tiny`` for what is below the type's normal numbers.
    Rows that see nothing count as 0, whatever stands in them; so do keys that nobody sees."""
    live_q, live_k = seen.any(1), seen.any(0)
    q = torch.where(live_q[:, None], q, torch.zeros_like(q))
    k, v = (torch.where(live_k[:, None], x, torch.zeros_like(x)) for x in (k, v))
    th = torch.tanh(scale * (q @ k.T) / cap) if cap else None
    s = (cap * th if cap else scale * (q @ k.T)) - slope * dist
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(1, keepdim=True) if s.shape[1] else torch.full((s.shape[0], 1), -math.inf, dtype=s.dtype)
    p = torch.exp(s - torch.where(live_q[:, None], m, torch.zeros_like(m)))
    l = p.sum(1, keepdim=True)
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    lse = torch.where(live_q, (m + torch.log(l))[:, 0], torch.full_like(l[:, 0], -math.inf)) / math.log(2.0)
    o = p @ v
    few = tiny * seen.double()
    o_off = (half * p + few) @ v.abs() + half * o.abs()
    if do is None:
        return (o, lse), (o_off,)
    do = torch.where(live_q[:, None], do, torch.zeros_like(do))
    inner = 1 - th * th if cap else torch.ones_like(p)
    ds = p * inner * (do @ v.T - (o * do).sum(1, keepdim=True)) * scale
    delta_off = (o_off * do.abs()).sum(1, keepdim=True)
    ds_off = half * ds.abs() + scale * p * inner * delta_off + few
    dq, dk, dv = ds @ k, ds.T @ q, p.T @ do
    return (o, lse, dq, dk, dv), (o_off, ds_off @ k.abs() + half * dq.abs(), ds_off.T @ q.abs(), (half * p + few).T @ do.abs())


def packed(q, k, v, cu_q, cu_k, scale, cap=0.0, slopes=None, window=None, doc_ids=None, prefix_lens=None, do=None, dtype=None):
    """o, lse [, dq, dk, dv] and their allowances for 16-bit type ``dtype`` (None: no roundings)."""
    half = torch.finfo(dtype).eps / 2 if dtype else 0.0
    tiny = torch.finfo(dtype).smallest_normal * half if dtype else 0.0
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    do = do.detach().double().cpu() if do is not None else None
    N, Hq, d = q.shape
    G = Hq // k.shape[1]
    o, lse = torch.zeros_like(q), torch.full((Hq, N), -math.inf, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    off = [torch.zeros_like(x) for x in (o, dq, dk, dv)]
    for b in range(len(cu_q) - 1):
        qs, ks = slice(int(cu_q[b]), int(cu_q[b + 1])), slice(int(cu_k[b]), int(cu_k[b + 1]))
        seen, dist = visible(qs.stop - qs.start, ks.stop - ks.start, window, doc_ids[ks].cpu() if doc_ids is not None else None,
                             int(prefix_lens[b]) if prefix_lens is not None else None)
        if not seen.numel():
            continue
        for h in range(Hq):
            g = h // G
            r, e = one_head(q[qs, h], k[ks, g], v[ks, g], seen, dist, scale, cap, float(slopes[h]) if slopes is not None else 0.0,
                            do[qs, h] if do is not None else None, half, tiny)
            o[qs, h], lse[h, qs], off[0][qs, h] = r[0], r[1], e[0]
            if do is not None:
                dq[qs, h], off[1][qs, h] = r[2], e[1]
                dk[ks, g] += r[3]
                dv[ks, g] += r[4]
                off[2][ks, g] += e[2]
                off[3][ks, g] += e[3]
    off[2] += half * dk.abs()
    off[3] += half * dv.abs()
    if do is None:
        return (o, lse), off[:1]
    return (o, lse, dq, dk, dv), off


def decoded(q, k, v, seq_len, row0, scale, cap=0.0, slopes=None, window=None, prefixes=None, dtype=None):
    """One token a sequence: o, lse [B, Hq] and o's allowance.  prefixes: for every sequence (k, v) rows in front of its own."""
    half = torch.finfo(dtype).eps / 2 if dtype else 0.0
    tiny = torch.finfo(dtype).smallest_normal * half if dtype else 0.0
    q, k, v = (x.double().cpu() for x in (q, k, v))
    B, Hq, d = q.shape
    G = Hq // k.shape[1]
    o, lse, off = torch.zeros_like(q), torch.full((B, Hq), -math.inf, dtype=torch.float64), torch.zeros_like(q)
    for b in range(B):
        n = int(seq_len[b])
        if n <= 0:
            continue
        rows = slice(int(row0[b]), int(row0[b]) + n)
        kb, vb = k[rows], v[rows]
        if prefixes is not None:
            kb, vb = torch.cat([prefixes[b][0].double().cpu(), kb]), torch.cat([prefixes[b][1].double().cpu(), vb])
        seen, dist = visible(1, kb.shape[0], window)
        for h in range(Hq):
            r, e = one_head(q[b : b + 1, h], kb[:, h // G], vb[:, h // G], seen, dist, scale, cap, float(slopes[h]) if slopes is not None else 0.0,
                            None, half, tiny)
            o[b, h], lse[b, h], off[b, h] = r[0][0], r[1][0], e[0][0]
    return (o, lse), off
