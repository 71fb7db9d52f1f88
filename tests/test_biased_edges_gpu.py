"""Attention with changed scores where a call is allowed but unusual.  Allowances as in test_biased_attn_gpu.py, where nothing else is said."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fsa.ops import biased_attention
from fsa_preview.ops import biased_decode_attention, shared_prefix_decode_attention
from oracle import biased_attn_oracle as orc
from test_biased_attn_gpu import BF16, DEV, check, cu_of, inputs, near, near_lse
from test_biased_decode_gpu import cache_of, i32


@pytest.mark.parametrize("G,front,groups", [(32, 9, 36), (4, 70, 33), (32, 130, 400), (1, 260, 40)])
def test_many_groups_behind_at_least_a_tile_of_sequences_without_one(G, front, groups):
    """More groups than a warp has lanes, and so many sequences in front of the first one that whole tiles lie there."""
    assert groups > 32 and front >= (128 // G) & ~3
    P, d = 20, 64
    lens = [1 + (7 * i) % 30 for i in range(front + groups + 2)]
    q, k, v, row0 = cache_of(lens, 1, G, d, BF16, 6)
    g = torch.Generator().manual_seed(7)
    pk, pv = (torch.randn(P * groups, 1, d, generator=g).to(BF16) for _ in range(2))
    o, lse = shared_prefix_decode_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(lens), i32(row0), pk.to(DEV), pv.to(DEV), cu_of([P] * groups).to(DEV),
                                            i32([front + i for i in range(groups + 1)]), max_len=30, max_prefix=P, softcap=20.0)
    mine = [(pk[P * (b - front) : P * (b - front + 1)], pv[P * (b - front) : P * (b - front + 1)]) if front <= b < front + groups else (pk[:0], pv[:0])
            for b in range(len(lens))]
    ref, off = orc.decoded(q, k, v, lens, row0, d ** -0.5, 20.0, None, None, mine, BF16)
    near(o, ref[0], off, "o")
    near_lse(lse, ref[1])


@pytest.mark.parametrize("Hk,G,d", [(1, 2, 64), (2, 1, 128)])
def test_prefixes_below_zero(Hk, G, d):
    """The smallest number in the sequence that begins at row 0: nobody sees the rows of another sequence."""
    lens = [90, 40, 130]
    q, k, v, do = inputs(lens, lens, Hk, G, d, BF16, 2)
    for prefix in ([-2 ** 31] * 3, [-1, 7, -2 ** 31]):
        check(q, k, v, do, lens, lens, 20.0, None, prefix=torch.tensor(prefix, dtype=torch.int32))


@pytest.mark.parametrize("cap", [1e4, 1e6, 1e8])
@pytest.mark.parametrize("d,dtype", [(64, BF16), (128, BF16)])
def test_a_cap_that_one_token_reaches(cap, d, dtype):
    """One token's scores are as large as a cap far above all the others': those get what they get without it."""
    lens, big = [130], 40
    q, k, v, do = inputs(lens, lens, 1, 2, d, dtype, 3)
    q[big], do[big] = q[big] * cap, 0.0
    cu = cu_of(lens)
    ref, off = orc.packed(q, k, v, cu, cu, d ** -0.5, cap, do=do, dtype=dtype)
    leaves = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    o, lse = biased_attention(*leaves, cu.to(DEV), softcap=cap)
    grads = torch.autograd.grad(o, leaves, do.to(DEV))
    rest = [t for t in range(lens[0]) if t != big]
    near(o.detach()[rest], ref[0][rest], off[0][rest], "o")
    near_lse(lse[:, rest], ref[1][:, rest])
    near(grads[0][rest], ref[2][rest], off[1][rest], "dq")
    # (without a dO the large one has no share in these)
    near(grads[1], ref[3], off[2], "dk")
    near(grads[2], ref[4], off[3], "dv")


@pytest.mark.parametrize("cap,scale", [(1e4, 0.1), (1e6, 0.1), (1e8, 0.1), (30.0, 1e-12), (1e20, 0.1)])
@pytest.mark.parametrize("d,G", [(64, 2), (128, 16)])
def test_decode_with_caps_far_above_the_scores(cap, scale, d, G):
    """Single tokens, behind shared rows too, and the same rows of a prefill: all of them right, so that they agree."""
    lens, P = [300, 0, 70], 200
    q, k, v, row0 = cache_of(lens, 1, G, d, BF16, 4)
    g = torch.Generator().manual_seed(5)
    pk, pv = (torch.randn(P, 1, d, generator=g).to(BF16) for _ in range(2))
    args, how = [x.to(DEV) for x in (q, k, v)] + [i32(lens), i32(row0)], dict(max_len=300, softcap=cap, sm_scale=scale)
    for mine, (o, lse) in ((None, biased_decode_attention(*args, **how)),
                           ([(pk, pv)] * 3, shared_prefix_decode_attention(*args, pk.to(DEV), pv.to(DEV), i32([0, P]), i32([0, 3]), **how))):
        ref, off = orc.decoded(q, k, v, lens, row0, scale, cap, None, None, mine, BF16)
        near(o, ref[0], off, "o")
        near_lse(lse, ref[1])
    for b in (0, 2):
        rows = slice(row0[b], row0[b] + lens[b])
        o1, lse1 = biased_attention(q[b : b + 1].to(DEV), k[rows].to(DEV), v[rows].to(DEV), i32([0, 1]), cu_seqlens_k=i32([0, lens[b]]), softcap=cap, sm_scale=scale)
        ref, off = orc.decoded(q, k, v, lens, row0, scale, cap, dtype=BF16)
        near(o1[0], ref[0][b], off[b], "o of a prefill")
        near_lse(lse1[:, 0], ref[1][b])
