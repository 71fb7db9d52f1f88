"""Attention with changed scores: the oracle against differences and against autograd, and what the operators refuse (no GPU needed)."""
import math

import pytest
import torch

from fsa.ops import biased_attention
from oracle import biased_attn_oracle as orc


def _case(cap, slope, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(n, 8, generator=g, dtype=torch.float64) for n in (5, 9, 9, 5))
    seen, dist = orc.visible(5, 9, window=4)
    return q, k, v, do, seen, dist, dict(scale=0.7, cap=cap, slope=slope)


@pytest.mark.parametrize("cap,slope", [(0.0, 0.0), (2.0, 0.0), (0.0, 0.3), (1.5, 0.2)])
def test_oracle_gradients_against_differences(cap, slope):
    q, k, v, do, seen, dist, how = _case(cap, slope)
    f = lambda q, k, v: float((orc.one_head(q, k, v, seen, dist, **how)[0][0] * do).sum())  # noqa: E731
    grads = orc.one_head(q, k, v, seen, dist, do=do, **how)[0][2:]
    h = 1e-6
    for n, (x, got) in enumerate(zip((q, k, v), grads)):
        for i, j in ((0, 0), (1, 3), (4, 7)):
            up, down = x.clone(), x.clone()
            up[i, j] += h
            down[i, j] -= h
            args = [q, k, v]
            a, b = (f(*(args[:n] + [y] + args[n + 1 :])) for y in (up, down))
            assert abs((a - b) / (2 * h) - float(got[i, j])) < 1e-7


def test_oracle_masks():
    seen, dist = orc.visible(3, 5, window=1)
    assert seen.tolist() == [[False, True, True, False, False], [False, False, True, True, False], [False, False, False, True, True]]
    assert dist[0].tolist() == [2, 1, 0, 1, 2]
    seen, _ = orc.visible(3, 3, prefix=2)
    assert seen.tolist() == [[True, True, False], [True, True, False], [True, True, True]]
    seen, _ = orc.visible(5, 5, ids=torch.tensor([1, 1, -1, 1, 1], dtype=torch.int32))
    assert seen.int().tolist() == [[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [0, 0, 0, 0, 0], [0, 0, 0, 1, 0], [0, 0, 0, 1, 1]]
    seen, _ = orc.visible(4, 2)                          # more queries than keys
    assert seen.tolist() == [[False, False], [False, False], [True, False], [True, True]]


def test_oracle_rows_that_see_nothing():
    q, k, v, do, seen, dist, how = _case(2.0, 0.1)
    seen[2] = False
    seen[:, 8] = False
    q[2], do[2], k[8], v[8] = math.nan, math.inf, math.nan, math.inf
    (o, lse, dq, dk, dv), _ = orc.one_head(q, k, v, seen, dist, do=do, **how)
    assert float(lse[2]) == -math.inf and all(bool(torch.isfinite(x).all()) for x in (o, dq, dk, dv))
    assert bool((o[2] == 0).all()) and bool((dk[8] == 0).all())


BF16 = torch.bfloat16


def _args(N=6, Nk=6, Hq=4, Hk=2, d=64, dtype=BF16):
    return [torch.zeros(N, Hq, d, dtype=dtype), torch.zeros(Nk, Hk, d, dtype=dtype), torch.zeros(Nk, Hk, d, dtype=dtype), torch.tensor([0, N], dtype=torch.int32)]


@pytest.mark.parametrize("what,change,error", [
    ("a type", dict(dtype=torch.float32), TypeError),
    ("heads", dict(Hq=3), ValueError),
    ("a head size", dict(d=256), ValueError),
    ("a head size", dict(d=80), ValueError),
    ("a group", dict(Hq=66, Hk=2), ValueError),
    ("lengths", dict(Nk=7), ValueError),
])
def test_refuses_shapes(what, change, error):
    with pytest.raises(error):
        biased_attention(*_args(**change))


@pytest.mark.parametrize("how,error", [
    (dict(softcap=-1.0), ValueError),
    (dict(softcap=math.inf), ValueError),
    (dict(softcap=math.nan), ValueError),
    (dict(sm_scale=0.0), ValueError),
    (dict(sm_scale=math.nan), ValueError),
    (dict(window_size=-1), ValueError),
    (dict(alibi_slopes=torch.zeros(3)), ValueError),
    (dict(alibi_slopes=torch.zeros(4, dtype=torch.float64)), TypeError),
    (dict(alibi_slopes=torch.zeros(4, requires_grad=True)), ValueError),
    (dict(doc_ids=torch.zeros(5, dtype=torch.int32)), ValueError),
    (dict(doc_ids=torch.zeros(6, dtype=torch.int64)), TypeError),
    (dict(prefix_lens=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(prefix_lens=torch.zeros(1, dtype=torch.int32), window_size=3), ValueError),
    (dict(prefix_lens=torch.zeros(1, dtype=torch.int32), doc_ids=torch.zeros(6, dtype=torch.int32)), ValueError),
    (dict(cu_seqlens_k=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(), ValueError),                                # no CUDA tensors
])
def test_refuses_arguments(how, error):
    with pytest.raises(error):
        biased_attention(*_args(), **how)


def test_refuses_other_types_of_lengths():
    a = _args()
    with pytest.raises(TypeError):
        biased_attention(*a[:3], a[3].long())
    with pytest.raises(ValueError):
        biased_attention(*a[:3], a[3][:1])
    with pytest.raises(TypeError):
        biased_attention(a[0], a[1].half(), a[2], a[3])
