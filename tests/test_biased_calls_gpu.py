"""Attention with changed scores at lengths where a kernel's blocks take several pieces of work each, with many sequences, at the ends of
its arguments' ranges, and in calls side by side.

Allowances as in test_biased_attn_gpu.py, with a slack of 1.2 instead of 1.05 for sums of up to n = 6000 terms: in 32 bits these are off by
n 2^-24 = 2^-11.4 of their terms' sizes at most, 0.18 of the half step 2^-9 that the allowance counts for every bf16 term."""
import math
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

from fsa.ops import biased_attention
from fsa_preview.ops import biased_decode_attention, shared_prefix_decode_attention
from oracle import biased_attn_oracle as orc
from test_biased_attn_gpu import BF16, DEV, check, cu_of, inputs, near, near_lse, slopes_of
from test_biased_decode_gpu import cache_of, check as check_decode, i32

INT_MAX = 2 ** 31 - 1


def roomy(got, ref, off, name):
    err = (got.double() - ref).abs()
    room = 1.2 * off + 2.0 ** -20 * float(ref.abs().max())
    assert bool((err <= room).all()), f"{name}: {float((err - room).max()):.3e} over the allowance"


@pytest.mark.parametrize("Hk,G,d,cap,alibi,how", [
    (8, 1, 128, 30.0, False, {}),                     # 47 K/V tiles and 8 heads: several pieces of work an SM, tiles cut
    (4, 4, 64, None, True, {}),
    (8, 2, 128, None, False, {"window": 700}),
    (4, 2, 128, 50.0, True, {"docs": 900}),
    (4, 1, 64, 20.0, True, {"prefix": 2500}),
    (1, 1, 128, 30.0, True, {}),                      # one head: o and dQ cut along the keys
    (1, 2, 64, None, False, {}),
    (1, 1, 64, 20.0, False, {"docs": 3500}),
    (1, 1, 128, None, True, {"window": 2900}),
])
def test_long(Hk, G, d, cap, alibi, how):
    N, Hq = 6000, Hk * G
    q, k, v, do = (x.to(DEV) for x in inputs([N], [N], Hk, G, d, BF16, N + G))
    ids = torch.div(torch.arange(N, dtype=torch.int32), how["docs"], rounding_mode="floor").int() if "docs" in how else None
    sl = slopes_of(Hq) if alibi else None
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    o, lse = biased_attention(*leaves, i32([0, N]), softcap=cap, alibi_slopes=None if sl is None else sl.to(DEV), window_size=how.get("window"),
                              doc_ids=None if ids is None else ids.to(DEV), prefix_lens=i32([how["prefix"]]) if "prefix" in how else None)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    seen, dist = (x.to(DEV) for x in orc.visible(N, N, how.get("window"), ids, how.get("prefix")))
    half = torch.finfo(BF16).eps / 2
    tiny = torch.finfo(BF16).smallest_normal * half
    for kh in range(Hk):
        sums = [0.0] * 4
        for h in range(kh * G, kh * G + G):
            ref, off = orc.one_head(*(x.double() for x in (q[:, h], k[:, kh], v[:, kh])), seen, dist, d ** -0.5, cap or 0.0, float(sl[h]) if alibi else 0.0,
                                    do[:, h].double(), half, tiny)
            roomy(o[:, h], ref[0], off[0], f"o of head {h}")
            near_lse(lse[h], ref[1].cpu())
            roomy(dq[:, h], ref[2], off[1], f"dq of head {h}")
            sums = [a + b for a, b in zip(sums, (ref[3], ref[4], off[2], off[3]))]
        # (dk and dv: the heads of a group are added in 32 bits, the sum is rounded once)
        roomy(dk[:, kh], sums[0], sums[2] + half * sums[0].abs(), f"dk of head {kh}")
        roomy(dv[:, kh], sums[1], sums[3] + half * sums[1].abs(), f"dv of head {kh}")


@pytest.mark.parametrize("how", [{}, {"window": 40}, {"docs": True}, {"prefix": True}])
def test_many_sequences(how):
    """More sequences than a block has threads, some without tokens, some with more keys than queries and the other way round."""
    lens = [3, 0, 130, 1, 17] * 130
    klens = [5, 2, 130, 0, 200] * 130
    q, k, v, do = inputs(lens, klens, 1, 2, 64, BF16, 9)
    ids = torch.div(torch.arange(sum(klens), dtype=torch.int32), 50, rounding_mode="floor").int() if "docs" in how else None
    prefix = torch.tensor([b % 140 for b in range(len(lens))], dtype=torch.int32) if "prefix" in how else None
    check(q, k, v, do, lens, klens, 20.0, slopes_of(2), window=how.get("window"), ids=ids, prefix=prefix)


@pytest.mark.parametrize("lens,klens", [([150, 40], [150, 40]), ([100, 20], [300, 10])])
def test_the_largest_window_and_prefix(lens, klens):
    """(The second sequence begins behind row 0: its first row and such a prefix are more than an int holds.)"""
    q, k, v, do = inputs(lens, klens, 1, 2, 128, BF16, 2)
    check(q, k, v, do, lens, klens, 20.0, None, window=INT_MAX)
    check(q, k, v, do, lens, klens, 20.0, None, prefix=torch.tensor([INT_MAX, INT_MAX], dtype=torch.int32))
    check(q, k, v, do, lens, klens, 20.0, None, prefix=torch.tensor([-1, -INT_MAX - 1], dtype=torch.int32))


@pytest.mark.parametrize("cap,scale", [(1e8, 0.1), (30.0, 1e-12), (1e20, 0.1)])
def test_caps_far_above_the_scores(cap, scale):
    lens = [90, 33]
    q, k, v, do = inputs(lens, lens, 1, 2, 64, BF16, 3)
    check(q, k, v, do, lens, lens, cap, scale=scale)


def test_a_cap_far_below_the_scores():
    """All scores are at the cap: their gradients are 0 but for the error of the tanh, 6e-7, which 1 - t^2 doubles: 2^-19 sm_scale sum_j p |dP - delta| |k|, and
    |dP - delta| is at most twice the largest |dP|, the sum over the p of a row is 1, and a key has up to 90 of them."""
    lens, scale = [90, 33], 0.1
    q, k, v, do = inputs(lens, lens, 1, 2, 64, BF16, 3)
    leaves = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    o, lse = biased_attention(*leaves, cu_of(lens).to(DEV), softcap=1e-6, sm_scale=scale)
    ref, off = orc.packed(q, k, v, cu_of(lens), cu_of(lens), scale, 1e-6, do=do, dtype=BF16)
    near(o.detach(), ref[0], off[0], "o")
    near_lse(lse, ref[1])
    dq, dk, dv = (x.double().cpu() for x in torch.autograd.grad(o, leaves, do.to(DEV)))
    most = 2.0 ** -18 * scale * float(torch.einsum("nhd,md->nhm", do.double(), v[:, 0].double()).abs().max())
    assert bool(((dq - ref[2]).abs() <= most * float(k.abs().max())).all())
    assert bool(((dk - ref[3]).abs() <= 2 * 90 * most * float(q.abs().max())).all())
    near(dv, ref[4], off[3], "dv")


def test_documents_with_fewer_keys_than_queries():
    """Tokens in front of a sequence's first row stand at negative places, in the first block's first row as well."""
    lens, klens = [400, 300, 5], [90, 350, 0]
    q, k, v, do = inputs(lens, klens, 1, 2, 64, BF16, 4)
    ids = torch.cat([torch.full((n,), i, dtype=torch.int32) for n, i in ((60, 3), (200, 1), (100, -1), (80, 1))])
    check(q, k, v, do, lens, klens, 20.0, slopes_of(2), ids=ids)


def test_sequences_in_front_of_the_first_group():
    """cu_group that begins behind 0: the sequences before it have no prefix either."""
    lens, prefixes = [70, 5, 300, 1, 40], [333, 64]
    q, k, v, row0 = cache_of(lens, 2, 2, 128, BF16, 6)
    g = torch.Generator().manual_seed(7)
    pk, pv = (torch.randn(sum(prefixes), 2, 128, generator=g).to(BF16) for _ in range(2))
    o, lse = shared_prefix_decode_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(lens), i32(row0), pk.to(DEV), pv.to(DEV), i32([0, 333, 397]),
                                            i32([1, 3, 4]), max_len=300, softcap=20.0)
    none, a, b = (pk[:0], pv[:0]), (pk[:333], pv[:333]), (pk[333:], pv[333:])
    ref, off = orc.decoded(q, k, v, lens, row0, 128 ** -0.5, 20.0, None, None, [none, a, a, b, none], BF16)
    near(o, ref[0], off, "o")
    near_lse(lse, ref[1])


def test_a_million_token_hint():
    """max_len far above what the cache holds: more chunks, the same rows."""
    lens = [200, 31]
    q, k, v, row0 = cache_of(lens, 1, 2, 64, BF16, 8)
    args = [q.to(DEV), k.to(DEV), v.to(DEV), i32(lens), i32(row0)]
    ref, off = orc.decoded(q, k, v, lens, row0, 64 ** -0.5, 0.0, None, None, None, BF16)
    for hint in (0, 1 << 20):
        o, lse = biased_decode_attention(*args, max_len=hint)
        near(o, ref[0], off, "o")
        near_lse(lse, ref[1])
    with pytest.raises(ValueError, match="not supported"):
        biased_decode_attention(*args, max_len=1 << 30)


def test_two_graphs_replayed_at_once():
    """Two captured training steps, each on its own stream, replayed together."""
    lens, Hk, G, d = [900, 333], 2, 2, 128
    cu = cu_of(lens).to(DEV)
    steps, graphs, held = [], [], []
    for seed in (1, 2):
        *leaves, do = (x.to(DEV) for x in inputs(lens, lens, Hk, G, d, BF16, seed))
        leaves = [x.requires_grad_() for x in leaves]

        def step(leaves=leaves, do=do):
            o, lse = biased_attention(*leaves, cu, softcap=30.0)
            return [o.detach(), lse, *torch.autograd.grad(o, leaves, do)]

        steps.append(step)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step())
    want = [s() for s in steps]
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for x in held[0] + held[1]:
            x.zero_()
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for h, w in zip(held, want) for a, b in zip(h, w))


def test_steps_one_behind_another_on_one_stream():
    """Layers in a row without a pause, each writing where the one before it was read: what a kernel that starts early may not overtake."""
    lens = [1500, 40]
    cu = cu_of(lens).to(DEV)
    q, k, v, do = (x.to(DEV) for x in inputs(lens, lens, 2, 2, 64, BF16, 5))

    def run():
        x, out = q, []
        for i in range(6):
            leaves = [t.detach().requires_grad_() for t in (x, k, v)]
            o, _ = biased_attention(*leaves, cu, softcap=10.0 + i)
            dq, dk, dv = torch.autograd.grad(o, leaves, do)
            out += [dq, dk, dv]
            x = (o.detach() * 2 + dq).contiguous()
        return out

    first = run()
    torch.cuda.synchronize()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_gradients_need_not_be_asked_for_all():
    lens = [100]
    q, k, v, do = (x.to(DEV) for x in inputs(lens, lens, 1, 2, 64, BF16, 1))
    cu = cu_of(lens).to(DEV)
    kk = k.clone().requires_grad_()
    o, _ = biased_attention(q, kk, v, cu, softcap=5.0)
    every = [x.clone().requires_grad_() for x in (q, k, v)]
    o2, _ = biased_attention(*every, cu, softcap=5.0)
    assert torch.equal(torch.autograd.grad(o, kk, do)[0], torch.autograd.grad(o2, every, do)[1])
    with torch.no_grad():
        assert torch.equal(biased_attention(*every, cu, softcap=5.0)[0], o)


_WITH_CHECKS = """
import torch
from fsa.ops import biased_attention
from fsa_preview.ops import biased_decode_attention
x = [torch.randn(70, 2, 64, device="cuda").bfloat16().requires_grad_() for _ in range(3)]
cu = torch.tensor([0, 70], dtype=torch.int32, device="cuda")
o, lse = biased_attention(*x, cu, softcap=5.0)
o.float().sum().backward()
n = torch.tensor([70], dtype=torch.int32, device="cuda")
d, _ = biased_decode_attention(x[0][-1:].detach(), x[1].detach(), x[2].detach(), n, n * 0, max_len=70, softcap=5.0)
assert (d[0] - o[-1]).abs().max() <= 2 ** -6 * o.abs().max()
print("read")
"""


def test_with_status_checks():
    """FSA_CHECK_STATUS=1: the status word is read behind every call."""
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "flash-sparse-attention_b200")
    r = subprocess.run([sys.executable, "-c", _WITH_CHECKS], env={**os.environ, "FSA_CHECK_STATUS": "1", "PYTHONPATH": root}, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "read" in r.stdout, r.stderr[-2000:]


def cut_bytes(q, k, cu, window):
    """Workspace of a forward whose K/V rows are cut into chunks; 0: they are not."""
    import ctypes

    from fsa._lib import lib

    n = ctypes.c_int64(-1)
    assert lib().fsa_biased_attn_fwd_bytes(q.shape[0], k.shape[0], cu.numel() - 1, q.shape[1], k.shape[1], q.shape[2], -1 if window is None else window,
                                           ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("score", [(None, False), (20.0, False), (None, True), (50.0, True)])
@pytest.mark.parametrize("lens,klens,Hk,G,d,dtype,how", [
    ([1], [3001], 1, 1, 128, BF16, {}),                                # one query
    ([5, 0, 33], [2500, 700, 3100], 2, 4, 128, BF16, {}),              # a sequence without queries
    ([40, 3, 100], [4000, 2, 60], 1, 3, 64, torch.float16, {}),        # chunks without rows; fewer keys than queries
    ([17, 64], [3000, 2000], 1, 8, 128, BF16, {"window": 1500}),
    ([130, 20], [2500, 1500], 1, 2, 64, BF16, {"docs": True}),
    ([300, 70], [2500, 2200], 1, 4, 128, BF16, {"prefix": [2400, 2199]}),
    ([1900], [1900], 1, 1, 128, BF16, {"prefix": [1500]}),
])
def test_few_queries_over_many_keys(score, lens, klens, Hk, G, d, dtype, how):
    """Forward with the K/V rows cut into chunks: masks that leave chunks empty, padding of NaN in the middle."""
    cap, alibi = score
    q, k, v, do = inputs(lens, klens, Hk, G, d, dtype, sum(klens))
    assert cut_bytes(q, k, cu_of(lens), how.get("window")) > 0
    ids = None
    if "docs" in how:
        ids = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in ((1, 300), (-1, 100), (2, 2100), (4, 700), (-3, 90), (5, 710))])
        k[ids < 0], v[ids < 0] = math.nan, math.inf
    prefix = torch.tensor(how["prefix"], dtype=torch.int32) if "prefix" in how else None
    check(q, k, v, do, lens, klens, cap, slopes_of(Hk * G) if alibi else None, window=how.get("window"), ids=ids, prefix=prefix)


def test_chunks_and_rows_behind_the_last_sequence():
    lens, klens, spare = [30, 11], [2600, 2100], 50
    q, k, v, _ = inputs(lens, klens, 2, 2, 128, BF16, 1)
    pad = lambda x: torch.cat([x, torch.full((spare, *x.shape[1:]), math.nan, dtype=x.dtype)]).to(DEV)  # noqa: E731
    qc, kc, vc = pad(q), pad(k), pad(v)
    assert cut_bytes(qc, kc, cu_of(lens), None) > 0
    o, lse = biased_attention(qc, kc, vc, cu_of(lens).to(DEV), cu_seqlens_k=cu_of(klens).to(DEV), softcap=30.0)
    ref, off = orc.packed(q, k, v, cu_of(lens), cu_of(klens), 128 ** -0.5, 30.0, dtype=BF16)
    n = sum(lens)
    near(o[:n], ref[0], off[0], "o")
    near_lse(lse[:, :n], ref[1])
    assert bool((o[n:] == 0).all()) and bool((lse[:, n:] == -math.inf).all())
    again = biased_attention(qc, kc, vc, cu_of(lens).to(DEV), cu_seqlens_k=cu_of(klens).to(DEV), softcap=30.0)
    assert torch.equal(again[0], o) and torch.equal(again[1], lse)


def test_a_verification_step_agrees_with_single_tokens():
    """Four drafted tokens after a cache in one call, and the same tokens one at a time over the cache: the rows agree to what P's rounding and o's make."""
    Hk, G, d, L = 2, 4, 128, 5000
    q, k, v, _ = (x.to(DEV) for x in inputs([4], [L], Hk, G, d, BF16, 12))
    o, lse = biased_attention(q, k, v, i32([0, 4]), cu_seqlens_k=i32([0, L]), softcap=40.0, alibi_slopes=slopes_of(8).to(DEV))
    for i in range(4):
        o1, lse1 = biased_decode_attention(q[i : i + 1], k, v, i32([L - 3 + i]), i32([0]), max_len=L, softcap=40.0, alibi_slopes=slopes_of(8).to(DEV))
        # each side: half a step 2^-9 of P (sums of |p v|, at most max |v|), and 2^-9 of o
        assert float((o[i] - o1[0]).abs().max()) <= 2 * 2.0 ** -8 * float(v.abs().max())
        assert float((lse[:, i] - lse1[0]).abs().max()) <= 2.0 ** -15


def test_many_groups():
    """More shared prefixes than a warp has lanes, some with no sequence, some of no rows."""
    prefixes = [100, 1, 0, 70, 333] * 9
    groups = [1, 0, 3, 2, 40] * 9
    lens = [(i * 7) % 50 + 1 for i in range(sum(groups) + 3)]
    check_decode(lens, 2, 4, 64, BF16, "both", prefixes=prefixes, groups=groups)


def test_many_groups_behind_sequences_without_one():
    lens, prefixes = [70, 5, 300, 1, 40] * 8, [90] * 36
    q, k, v, row0 = cache_of(lens, 1, 4, 64, BF16, 6)
    g = torch.Generator().manual_seed(7)
    pk, pv = (torch.randn(sum(prefixes), 1, 64, generator=g).to(BF16) for _ in range(2))
    cg = [3 + i for i in range(37)]         # sequences 3 .. 38, one a group
    o, lse = shared_prefix_decode_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(lens), i32(row0), pk.to(DEV), pv.to(DEV), cu_of(prefixes).to(DEV), i32(cg),
                                            max_len=300, softcap=20.0)
    mine = [(pk[(b - 3) * 90 : (b - 2) * 90], pv[(b - 3) * 90 : (b - 2) * 90]) if 3 <= b < 39 else (pk[:0], pv[:0]) for b in range(len(lens))]
    ref, off = orc.decoded(q, k, v, lens, row0, 64 ** -0.5, 20.0, None, None, mine, BF16)
    near(o, ref[0], off, "o")
    near_lse(lse, ref[1])


def test_many_sequences_of_one_token():
    lens = [1] * 700 + [0] * 40 + [300] + [1] * 50
    q, k, v, do = inputs(lens, lens, 2, 4, 64, BF16, 10)
    check(q, k, v, do, lens, lens, 20.0, slopes_of(8))


@pytest.mark.parametrize("score", [(20.0, False), (50.0, True)])
@pytest.mark.parametrize("lens,klens", [([400, 1, 250], [400, 1, 250]), ([60, 7, 300], [500, 90, 300])])
@pytest.mark.parametrize("window", [0, 33, 150])
def test_documents_within_a_window(score, lens, klens, window):
    cap, alibi = score
    q, k, v, do = inputs(lens, klens, 1, 4, 128, BF16, window + len(klens))
    g = torch.Generator().manual_seed(window)
    ids = torch.cumsum((torch.rand(sum(klens), generator=g) < 0.02).int(), 0).to(torch.int32)
    ids[100:130] = -1
    check(q, k, v, do, lens, klens, cap, slopes_of(4) if alibi else None, window=window, ids=ids)


@pytest.mark.parametrize("prefix", [None, [300, 20]])
def test_scores_that_grow_with_the_distance(prefix):
    """Negative slopes: the furthest keys weigh most, so a row's maximum rises tile after tile."""
    lens = [400, 130]
    q, k, v, do = inputs(lens, lens, 2, 2, 64, BF16, 13)
    check(q, k, v, do, lens, lens, None, torch.tensor([-0.05, 0.0, -0.01, 0.05]), prefix=None if prefix is None else torch.tensor(prefix, dtype=torch.int32))


def test_capture_beside_a_live_graph_of_the_same_leaves():
    """Refused before anything is captured; once the eager graph is gone, the capture holds forward and backward."""
    lens = [100]
    q, k, v, do = (x.to(DEV) for x in inputs(lens, lens, 1, 2, 64, BF16, 14))
    cu = cu_of(lens).to(DEV)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o, _ = biased_attention(*leaves, cu, softcap=5.0)
    want = o.detach().clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="leaf of this capture"):
        with torch.cuda.graph(graph):
            biased_attention(*leaves, cu, softcap=5.0)
    del o
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, _ = biased_attention(*leaves, cu, softcap=5.0)
        grads = torch.autograd.grad(o, leaves, do)
    graph.replay()
    assert torch.equal(o.detach(), want) and all(bool(torch.isfinite(x).all()) for x in grads)


def test_offsets_beyond_32_bits():
    """2.3e9 elements of q: the last sequences get what they get alone, bit for bit.  dk and dv but for the order of their sums: alone, a K/V tile's 25 row tiles
    are cut into four parts that are added up (items of 8 row tiles at least, 740 wanted), among 1400 sequences they are not.  Sums of n = 3200 terms in 32 bits in two orders differ by
    2 n 2^-24 = 2^-11.4 of the sum of their sizes at most, which for terms of random signs is 0.8 n / 4 sqrt(n) = 11 times the largest of some thousand such sums: 2^-7.9
    of that; and then by one step of bf16, 2^-7 of the value."""
    L, B, Hk, G, d = 100, 1400, 4, 32, 128
    N, Hq = L * B, Hk * G
    assert N * Hq * d > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(3)
    mk = lambda h: torch.randn(N, h, d, device=DEV, dtype=BF16, generator=g)  # noqa: E731
    q, k, v, do = mk(Hq), mk(Hk), mk(Hk), mk(Hq)
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV) * L
    sl = slopes_of(Hq).to(DEV)

    def step(q, k, v, do, cu):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        o, lse = biased_attention(*leaves, cu, softcap=20.0, alibi_slopes=sl)
        return [o.detach(), lse.T, *torch.autograd.grad(o, leaves, do)]

    whole = step(q, k, v, do, cu)
    n = 40 * L          # (more than 32 sequences: the same order of work)
    alone = step(q[-n:], k[-n:], v[-n:], do[-n:], cu[:41])
    for name, a, b in zip(("o", "lse", "dq", "dk", "dv"), whole, alone):
        a = a[-n:]
        if name in ("dk", "dv"):
            x, y = a.double(), b.double()
            assert bool(((x - y).abs() <= 2.0 ** -7 * y.abs() + 2.0 ** -7.9 * float(y.abs().max())).all()), name
        else:
            assert torch.equal(a, b), name


def test_a_cache_beyond_32_bits():
    rows, Hk, G, d, lens = 4_300_000, 4, 4, 128, [3000, 17]
    assert rows * Hk * d > 2 ** 31
    k = torch.zeros(rows, Hk, d, device=DEV, dtype=BF16)
    v = torch.zeros_like(k)
    qs, kc, vc, row0 = cache_of(lens, Hk, G, d, BF16, 15)
    at = rows - kc.shape[0]
    k[at:], v[at:] = kc.to(DEV), vc.to(DEV)
    how = dict(max_len=3000, softcap=20.0)
    far = biased_decode_attention(qs.to(DEV), k, v, i32(lens), i32([r + at for r in row0]), **how)
    near_ = biased_decode_attention(qs.to(DEV), kc.to(DEV), vc.to(DEV), i32(lens), i32(row0), **how)
    assert torch.equal(far[0], near_[0]) and torch.equal(far[1], near_[1]) and bool(torch.isfinite(far[0]).all())
