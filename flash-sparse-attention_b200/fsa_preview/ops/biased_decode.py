"""One new token of every sequence with changed scores (capped by a tanh, biased by distance) over a K/V cache, and the same for
batches whose sequences continue a prefix that they share: the single-token forms of ``fsa.ops.biased_attention``.

The reference has no such operators; they stand next to the decode operators of ``fsa_preview.ops.decode`` and read the same
caches (``DecodeCache.k``, ``.v``, ``.seq_len``, ``.seq_row0``).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from fsa._host import host

__all__ = ["biased_decode_attention", "shared_prefix_decode_attention"]


def _window(window_size: Optional[int]) -> int:
    if window_size is None:
        return -1
    if window_size < 0:
        raise ValueError(f"window_size has to be 0 or more (or None), got {window_size}")
    return int(window_size)


def biased_decode_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    seq_len: torch.Tensor,
    seq_row0: torch.Tensor,
    *,
    max_len: int,
    sm_scale: Optional[float] = None,
    softcap: Optional[float] = None,
    alibi_slopes: Optional[torch.Tensor] = None,
    window_size: Optional[int] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of the last token of every sequence over its rows of a cache: what ``biased_attention`` gives that row.

    Args:
        q: ``[batch, num_q_heads, head_dim]`` bf16/fp16, head_dim 64 or 128
        k, v: cache rows ``[rows, num_kv_heads, head_dim]``, up to 32 query heads a kv head; read in place
        seq_len: ``[batch]`` int32: tokens of every sequence, the new one included (its K and V rows are in the cache).  0: an
            idle place of the batch
        seq_row0: ``[batch]`` int32: cache row of every sequence's first token
        max_len: how long the longest sequence is (host integer): by it the work is cut.  Longer ones are read all the same
        sm_scale: defaults to ``1/sqrt(head_dim)``
        softcap: cap of the scores; None (or 0): none
        alibi_slopes: ``[num_q_heads]`` float32, what a score loses for each token of distance
        window_size: W: only the last W + 1 tokens are seen
    Returns:
        ``o [batch, num_q_heads, head_dim]`` and its log-sum-exp ``[batch, num_q_heads]`` in log2 units; 0 and -inf at idle places.

    Rows behind a sequence may hold anything, NaN included; a NaN (or +infinity) among a sequence's scores gives NaN in o and lse.  No synchronisation: a CUDA graph can hold the call.
    """
    return host().biased_decode(q, k, v, seq_len, seq_row0, None, None, None, None, alibi_slopes, q.shape[-1] ** -0.5 if sm_scale is None else float(sm_scale),
                                0.0 if softcap is None else float(softcap), _window(window_size), int(max_len), 0)


def shared_prefix_decode_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    seq_len: torch.Tensor,
    seq_row0: torch.Tensor,
    prefix_k: torch.Tensor,
    prefix_v: torch.Tensor,
    cu_prefix: torch.Tensor,
    cu_group: torch.Tensor,
    *,
    max_len: int,
    max_prefix: Optional[int] = None,
    sm_scale: Optional[float] = None,
    softcap: Optional[float] = None,
    alibi_slopes: Optional[torch.Tensor] = None,
    window_size: Optional[int] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``biased_decode_attention`` for sequences that continue shared prefixes (many answers to one question, requests behind one
    system prompt): every prefix is read once for all sequences that share it.

    Args (besides those of ``biased_decode_attention``):
        seq_len: ``[batch]`` int32: every sequence's OWN tokens, behind its prefix, the new one included.  0: an idle place
        prefix_k, prefix_v: the prefixes' rows, one prefix after the other ``[rows, num_kv_heads, head_dim]``
        cu_prefix: ``[num_prefixes + 1]`` int32: where the prefixes begin in prefix_k
        cu_group: ``[num_prefixes + 1]`` int32: sequences ``cu_group[i] .. cu_group[i + 1] - 1`` continue prefix i (sequences in front of
            the first and behind the last group have no prefix)
        max_prefix: how long the longest prefix is (host integer; all of prefix_k's rows, if not given)
    Distances, and window_size, count from the beginning of the prefix: the new token stands at place
    ``len(prefix) + seq_len[b] - 1``.
    """
    return host().biased_decode(q, k, v, seq_len, seq_row0, prefix_k, prefix_v, cu_prefix, cu_group, alibi_slopes,
                                q.shape[-1] ** -0.5 if sm_scale is None else float(sm_scale), 0.0 if softcap is None else float(softcap), _window(window_size),
                                int(max_len), prefix_k.shape[0] if max_prefix is None else int(max_prefix))
