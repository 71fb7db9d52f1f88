"""One new token a sequence with changed scores, over a cache and over shared prefixes, against the definition in 64 bits.  Allowances
as in test_biased_attn_gpu.py: P is rounded once before it is multiplied, the result once."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fsa.ops import biased_attention
from fsa_preview.ops import biased_decode_attention, shared_prefix_decode_attention
from oracle import biased_attn_oracle as orc
from test_biased_attn_gpu import BF16, DEV, FP16, SCORES, cu_of, near, near_lse, slopes_of


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cache_of(lens, Hk, G, d, dtype, seed, spare=3, qsize=2.0):
    """A cache of NaN in which every sequence's rows stand somewhere, in another order than the batch's."""
    g = torch.Generator().manual_seed(seed)
    mk = lambda n, h, s=1.0: (torch.randn(n, h, d, generator=g) * s).to(dtype)  # noqa: E731
    k = torch.full((sum(lens) + spare * (len(lens) + 1), Hk, d), math.nan, dtype=dtype)
    v = torch.full_like(k, math.inf)
    row0, at = [0] * len(lens), spare
    for b in reversed(range(len(lens))):
        row0[b] = at
        k[at : at + lens[b]], v[at : at + lens[b]] = mk(lens[b], Hk), mk(lens[b], Hk)
        at += lens[b] + spare
    return mk(len(lens), Hk * G, qsize), k, v, row0


def check(lens, Hk, G, d, dtype, score, window=None, prefixes=None, groups=None, hints=(None, None), seed=1, qsize=2.0):
    cap, alibi = SCORES[score]
    q, k, v, row0 = cache_of([max(n, 0) for n in lens], Hk, G, d, dtype, seed, qsize=qsize)
    sl = slopes_of(Hk * G) if alibi else None
    how = dict(softcap=cap, alibi_slopes=None if sl is None else sl.to(DEV), window_size=window, max_len=hints[0] or max([1] + lens))
    args = [q.to(DEV), k.to(DEV), v.to(DEV), i32(lens), i32(row0)]
    mine = None
    if prefixes is None:
        o, lse = biased_decode_attention(*args, **how)
    else:
        g = torch.Generator().manual_seed(seed + 1)
        pk, pv = (torch.randn(sum(prefixes), Hk, d, generator=g).to(dtype) for _ in range(2))
        cp, cg = cu_of(prefixes), cu_of(groups)
        of = [i for i, n in enumerate(groups) for _ in range(n)] + [None] * (len(lens) - sum(groups))
        mine = [(pk[:0], pv[:0]) if i is None else (pk[cp[i] : cp[i + 1]], pv[cp[i] : cp[i + 1]]) for i in of]
        o, lse = shared_prefix_decode_attention(*args, pk.to(DEV), pv.to(DEV), cp.to(DEV), cg.to(DEV), max_prefix=hints[1], **how)
    ref, off = orc.decoded(q, k, v, lens, row0, d ** -0.5, cap or 0.0, sl, window, mine, dtype)
    assert o.dtype == dtype and lse.dtype == torch.float32
    near(o, ref[0], off, "o")
    near_lse(lse, ref[1])


@pytest.mark.parametrize("score", list(SCORES))
@pytest.mark.parametrize("lens,Hk,G,d,dtype", [
    ([1], 1, 1, 64, BF16),
    ([700, 1, 64, 65, 0, 300], 2, 4, 128, BF16),         # an idle place; rows behind every sequence are NaN
    ([129, 1000], 1, 8, 64, FP16),
    ([333, 90], 2, 11, 128, FP16),                       # heads in the upper half of the MMA's rows
    ([200, 17], 1, 17, 64, BF16),                        # ... and in a second CTA
    ([150], 1, 32, 128, BF16),
    ([40, 3] * 20, 2, 2, 128, BF16),
])
def test_decode(score, lens, Hk, G, d, dtype):
    check(lens, Hk, G, d, dtype, score)


@pytest.mark.parametrize("score", list(SCORES))
@pytest.mark.parametrize("window", [0, 1, 63, 100, 5000])
def test_decode_window(score, window):
    check([700, 1, 64, 101, 0, 300], 2, 4, 128, BF16, score, window=window)


def test_decode_hints_do_not_change_what_is_read():
    for hint in (1, 64, 100, 5000):
        check([700, 1, 300], 2, 4, 128, BF16, "both", hints=(hint, None))
        check([700, 1, 300], 2, 4, 64, BF16, "cap", prefixes=[500, 33], groups=[2, 1], hints=(hint, hint))


def test_decode_saturated_cap():
    check([300, 7], 2, 4, 128, BF16, "cap", qsize=40.0)
    check([30, 7], 2, 4, 64, FP16, "cap", prefixes=[400], groups=[2], qsize=40.0)


@pytest.mark.parametrize("score", list(SCORES))
@pytest.mark.parametrize("prefixes,groups,lens,Hk,G,d,dtype", [
    ([500], [3], [1, 77, 130], 2, 4, 128, BF16),
    ([64], [1], [1], 1, 1, 64, FP16),
    ([1, 0, 700], [2, 3, 2], [5, 1, 9, 64, 2, 300, 1], 2, 2, 64, BF16),            # a prefix of one row, and one of none
    ([333], [70], [1 + i % 5 for i in range(70)], 1, 4, 128, FP16),                 # three tiles of 32 sequences
    ([200, 129], [3, 0], [4, 0, 6, 70, 0, 12], 1, 3, 128, BF16),                    # an empty group, idle places, sequences without a prefix
    ([260], [9], [3] * 9, 1, 20, 64, BF16),
    ([130], [5], [0] * 5, 1, 2, 128, BF16),                                         # nobody is at work
    ([90 + i for i in range(35)], [1] * 35, [2] * 35, 1, 2, 64, FP16),              # more groups than are ranked
])
def test_shared_prefix(score, prefixes, groups, lens, Hk, G, d, dtype):
    check(lens, Hk, G, d, dtype, score, prefixes=prefixes, groups=groups)


@pytest.mark.parametrize("window", [0, 10, 76, 200, 900])
@pytest.mark.parametrize("score", list(SCORES))
def test_shared_prefix_window(score, window):
    """Windows that end in a sequence's own rows, in the prefix, and before it."""
    check([1, 77, 130, 12], 2, 4, 128, BF16, score, window=window, prefixes=[500, 40], groups=[3, 1])


def test_prefix_rows_of_a_larger_buffer():
    """Rows behind the last prefix hold NaN; prefix rows and cache are views of one buffer of K and V."""
    Hk, G, d, P = 2, 4, 128, 150
    g = torch.Generator().manual_seed(2)
    both = torch.randn(600, 2, Hk, d, generator=g).to(BF16)
    both[P:200] = math.nan
    q = torch.randn(2, Hk * G, d, generator=g).to(BF16)
    lens, row0 = [100, 260], [200, 320]
    kv = both.to(DEV)
    k, v = kv[:, 0], kv[:, 1]
    o, lse = shared_prefix_decode_attention(q.to(DEV), k, v, i32(lens), i32(row0), k[:200], v[:200], i32([0, P]), i32([0, 2]), max_len=260, softcap=20.0)
    ref, off = orc.decoded(q, both[:, 0], both[:, 1], lens, row0, d ** -0.5, 20.0, prefixes=[(both[:P, 0], both[:P, 1])] * 2, dtype=BF16)
    near(o, ref[0], off, "o")
    near_lse(lse, ref[1])


def test_empty_batch():
    z = torch.zeros(4, 2, 64, dtype=BF16, device=DEV)
    o, lse = biased_decode_attention(torch.zeros(0, 4, 64, dtype=BF16, device=DEV), z, z, i32([]), i32([]), max_len=0)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_decode_from_a_graph_and_on_another_stream():
    lens, Hk, G, d = [300, 41], 2, 4, 128
    q, k, v, row0 = cache_of([400, 400], Hk, G, d, BF16, 3)
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(x.shape, generator=g).to(BF16).to(DEV) for x in (k, v))
    q, n, r = q.to(DEV), i32(lens), i32(row0)
    pk, pv, cp, cg = k[:200], v[:200], i32([0, 200]), i32([0, 2])
    run = lambda: shared_prefix_decode_attention(q, k, v, n, r, pk, pv, cp, cg, max_len=400, softcap=30.0, alibi_slopes=sl)  # noqa: E731
    sl = slopes_of(Hk * G).to(DEV)
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    with torch.cuda.graph(graph2):
        held2 = run()
    n += 1                                       # the next token, by the device-side lengths
    q.mul_(0.5)
    graph.replay()
    graph2.replay()
    want = run()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, held, held2)) and not torch.equal(want[0], first[0])


@pytest.mark.parametrize("score", list(SCORES))
def test_prefill_and_sampling_together(score):
    """A prompt is prefilled, then four answers to it are sampled: every decoded token gets what the packed operator gives the last
    row of prompt + answer, up to both sides' roundings."""
    cap, alibi = SCORES[score]
    Hk, G, d, P, steps, n = 2, 4, 128, 300, 5, 4
    Hq, sl = Hk * G, slopes_of(Hk * G).to(DEV) if alibi else None
    g = torch.Generator().manual_seed(11)
    mk = lambda rows, h: torch.randn(rows, h, d, generator=g).to(BF16).to(DEV)  # noqa: E731
    q, pk, pv = mk(P, Hq), mk(P, Hk), mk(P, Hk)
    o, _ = biased_attention(q, pk, pv, i32([0, P]), softcap=cap, alibi_slopes=sl)
    assert torch.isfinite(o).all()
    ck, cv = mk(n * steps, Hk), mk(n * steps, Hk)
    row0 = i32([steps * b for b in range(n)])
    for t in range(1, steps + 1):
        new = mk(n, Hq)
        got, lse = shared_prefix_decode_attention(new, ck, cv, i32([t] * n), row0, pk, pv, i32([0, P]), i32([0, n]), max_len=steps, softcap=cap,
                                                  alibi_slopes=sl)
        keys = torch.cat([torch.cat([pk, ck[steps * b : steps * b + t]]) for b in range(n)])
        vals = torch.cat([torch.cat([pv, cv[steps * b : steps * b + t]]) for b in range(n)])
        want, lse2 = biased_attention(new, keys, vals, i32(list(range(n + 1))), cu_seqlens_k=i32([b * (P + t) for b in range(n + 1)]), softcap=cap,
                                      alibi_slopes=sl)
        # both round P (2^-8 of |v| <= 4.5 weighted by p: below 2^-8) and the result
        assert float((got.float() - want.float()).abs().max()) <= 2 * (2.0 ** -8 + 2.0 ** -8 * float(want.abs().max()))
        assert float((lse.t() - lse2).abs().max()) <= 2.0 ** -15
