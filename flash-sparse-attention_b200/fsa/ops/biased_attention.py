"""Attention with changed scores over packed sequences, for training and prefill: scores capped by a tanh, biased by distance
(ALiBi), under causal, window, document and prefix masks.

    s = sm_scale q.k;   s = softcap tanh(s / softcap);   s = s - slope_h |t - j|;   o = softmax(s over the visible j) v

The reference has no such operator; it stands next to the sliding-window branch (``fsa.ops.range_attention``), with kernels of
its own.  One token of every sequence over a K/V cache: ``fsa_preview.ops.biased_decode``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from fsa._host import host

__all__ = ["biased_attention"]


def biased_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    cu_seqlens_k: Optional[torch.Tensor] = None,
    sm_scale: Optional[float] = None,
    softcap: Optional[float] = None,
    alibi_slopes: Optional[torch.Tensor] = None,
    window_size: Optional[int] = None,
    doc_ids: Optional[torch.Tensor] = None,
    prefix_lens: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention with changed scores, differentiable in q, k and v (once, in backward mode: forward-mode tangents and second derivatives are refused).

    Args:
        q: ``[total_len, num_q_heads, head_dim]`` bf16/fp16, head_dim 64 or 128
        k, v: ``[total_kv_len, num_kv_heads, head_dim]``, up to 32 query heads a kv head
        cu_seqlens: ``[batch + 1]`` int32, 0 first, where the sequences begin in q (and in k and v, unless cu_seqlens_k is given)
        cu_seqlens_k: ``[batch + 1]`` int32: where they begin in k and v (rows in front of the first are nobody's).  The queries of a sequence are its last tokens, as in
            a chunked prefill: query i of Lq stands at place ``t = Lk - Lq + i`` of the Lk keys (and sees none where t < 0)
        sm_scale: defaults to ``1/sqrt(head_dim)``
        softcap: cap of the scores; None (or 0): none
        alibi_slopes: ``[num_q_heads]`` float32, what a score loses for each token of distance; no gradient
        window_size: W: a token at place t sees the keys ``t - W <= j <= t``
        doc_ids: ``[total_kv_len]`` int32: a token sees only keys of its own document, the stretch of equal ids that it stands in.
            Negative: padding, which sees nothing and which nobody sees
        prefix_lens: ``[batch]`` int32: the first prefix_lens[b] keys of sequence b are seen by all its tokens (a prefix LM);
            not together with window_size or doc_ids
    Returns:
        ``o [total_len, num_q_heads, head_dim]`` and its log-sum-exp ``[num_q_heads, total_len]`` in log2 units (not
        differentiable).  A token that sees nothing, and rows behind the last sequence, get 0 and -inf.

    k and v rows that no token sees, and q rows of tokens that see nothing (and their gradients), may hold anything, NaN
    included.  What is seen and not a number goes on as in the formula: a token whose scores hold NaN (or +infinity) gets NaN in o and lse, and so
    do the gradients that it has a share in.  Gradients are the same bit for bit from run to run.  A CUDA graph can hold the call and its backward; while one is
    captured, no graph made on another stream may hold q, k or v as a leaf (RuntimeError).
    """
    if window_size is not None and window_size < 0:
        raise ValueError(f"window_size has to be 0 or more (or None), got {window_size}")
    return host().biased_attention(q, k, v, cu_seqlens, cu_seqlens_k, alibi_slopes, doc_ids, prefix_lens,
                                   q.shape[-1] ** -0.5 if sm_scale is None else float(sm_scale), 0.0 if softcap is None else float(softcap),
                                   -1 if window_size is None else int(window_size))
