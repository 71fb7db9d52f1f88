"""Attention with changed scores where a call is allowed but unusual.  Allowances as in test_biased_attn_gpu.py, where nothing else is said."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fsa.ops import biased_attention
from fsa_preview.ops import biased_decode_attention, shared_prefix_decode_attention
from oracle import biased_attn_oracle as orc
from test_biased_attn_gpu import BF16, DEV, check, cu_of, inputs, near, near_lse, slopes_of
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


SCORES_OF = [(None, False), (20.0, False), (None, True), (50.0, True)]


def same_where_finite(o, lse, ref, ref_lse, off):
    """NaN where the definition has NaN, and only there; the rest as everywhere.  o [rows, heads, d], lse and ref_lse [rows, heads]."""
    nan = torch.isnan(ref_lse)
    o, lse = o.detach().cpu(), lse.detach().cpu()
    assert torch.equal(torch.isnan(lse), nan), "lse"
    assert torch.equal(torch.isnan(o).all(-1), nan) and torch.equal(torch.isnan(o).any(-1), nan), "o"
    near(o[~nan], ref[~nan], off[~nan], "o")
    near_lse(lse[~nan], ref_lse[~nan])


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("cap,alibi", SCORES_OF)
@pytest.mark.parametrize("lens,klens,at,d,dtype", [
    ([200, 70], [200, 70], 130, 128, BF16),
    ([200, 70], [200, 70], 131, 64, torch.float16),
    ([6, 3], [3000, 2500], 1000, 128, BF16),             # cut along the keys: in one chunk of many
    ([6, 3], [3000, 2500], 2998, 64, BF16),              # seen by the sequence's last tokens only
])
def test_what_is_seen_and_not_a_number(lens, klens, at, d, dtype, cap, alibi, bad):
    """One number of a key that is seen: exactly the tokens whose softmax has no value get NaN, in o and lse, however the work is cut."""
    Hk, G = 2, 2
    q, k, v, _ = inputs(lens, klens, Hk, G, d, dtype, 9)
    k[at, 1, 5] = bad
    q[:, :, 5] = torch.where(q[:, :, 5] == 0, torch.ones_like(q[:, :, 5]), q[:, :, 5])
    cu, cuk = cu_of(lens), cu_of(klens)
    sl = slopes_of(Hk * G) if alibi else None
    how = dict(softcap=cap, alibi_slopes=None if sl is None else sl.to(DEV), cu_seqlens_k=cuk.to(DEV))
    o, lse = biased_attention(q.to(DEV), k.to(DEV), v.to(DEV), cu.to(DEV), **how)
    ref, off = orc.packed(q, k, v, cu, cuk, d ** -0.5, cap or 0.0, sl, dtype=dtype)
    if bad == bad and cap:                  # the cap makes numbers of infinite scores
        assert not torch.isnan(ref[1]).any()
    else:
        assert torch.isnan(ref[1]).any() and not torch.isnan(ref[1][:G]).any()
    same_where_finite(o, lse.T, ref[0], ref[1].T, off[0])


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("cap,alibi", SCORES_OF)
@pytest.mark.parametrize("where", ["own", "many", "prefix", "q"])
def test_decode_of_what_is_not_a_number(where, cap, alibi, bad):
    Hk, G, d, P = 2, 4, 128, 200
    lens = [700, 1, 130]
    q, k, v, row0 = cache_of(lens, Hk, G, d, BF16, 8)
    g = torch.Generator().manual_seed(5)
    pk, pv = (torch.randn(P, Hk, d, generator=g).to(BF16) for _ in range(2))
    if where == "own":
        k[row0[0] + 400, 1, 5] = bad
    elif where == "many":                   # all keys of some warps and chunks: with infinity, scores of -infinity for the heads whose q is negative there
        k[row0[0] + 100 : row0[0] + 690, 1, 5] = bad
    elif where == "prefix":
        pk[77, 1, 5] = bad
    elif bad == bad:
        return                              # (infinity in q: infinite scores of both signs)
    else:
        q[2, 3, 9] = bad
    sl = slopes_of(Hk * G) if alibi else None
    how = dict(max_len=700, softcap=cap, alibi_slopes=None if sl is None else sl.to(DEV))
    args = [x.to(DEV) for x in (q, k, v)] + [i32(lens), i32(row0)]
    for mine, (o, lse) in ((None, biased_decode_attention(*args, **how)),
                           ([(pk, pv)] * 3, shared_prefix_decode_attention(*args, pk.to(DEV), pv.to(DEV), i32([0, P]), i32([0, 3]), **how))):
        ref, off = orc.decoded(q, k, v, lens, row0, d ** -0.5, cap or 0.0, sl, None, mine, BF16)
        same_where_finite(o, lse, ref[0], ref[1], off)


@pytest.mark.parametrize("cap,alibi", SCORES_OF)
@pytest.mark.parametrize("lens,d", [([300], 128), ([4000], 64)])
def test_gradients_of_what_is_not_a_number(lens, d, cap, alibi):
    """A NaN in one token's q reaches its own dq and the dk and dv of every key that it sees; the other tokens' dq are what they are without it (not bit for
    bit: which of the two forms of the tanh, each off by 6e-7, a row takes its warp decides)."""
    t0, n = 170, lens[0]
    q, k, v, do = inputs(lens, lens, 1, 1, d, BF16, 10)
    sl, cu = slopes_of(1) if alibi else None, cu_of(lens)
    ref, off = orc.packed(q, k, v, cu, cu, d ** -0.5, cap or 0.0, sl, do=do, dtype=BF16)
    q[t0, 0, 3] = math.nan
    leaves = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    o, _ = biased_attention(*leaves, cu.to(DEV), softcap=cap, alibi_slopes=None if sl is None else sl.to(DEV))
    dq, dk, dv = torch.autograd.grad(o, leaves, do.to(DEV))
    assert bool(torch.isnan(dq[t0]).all()) and bool(torch.isnan(dk[: t0 + 1, 0, 3]).all()) and bool(torch.isnan(dv[: t0 + 1]).all())
    rest = [t for t in range(n) if t != t0]
    near(dq[rest], ref[2][rest], off[1][rest], "dq")
    near(dv[t0 + 1 :], ref[4][t0 + 1 :], off[3][t0 + 1 :], "dv")


def test_gradients_of_tokens_that_saw_a_key_that_is_not_a_number():
    lens, at = [260], 130
    q, k, v, do = inputs(lens, lens, 1, 2, 128, BF16, 11)
    k[at, 0, 0] = math.nan
    leaves = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    o, _ = biased_attention(*leaves, cu_of(lens).to(DEV), softcap=20.0)
    dq, dk, dv = torch.autograd.grad(o, leaves, do.to(DEV))
    assert bool(torch.isnan(dq[at:]).all()) and bool(torch.isnan(dk).all()) and bool(torch.isnan(dv).all())


def spread(x, dtype):
    """Variance of a value's rounding error, at most: uniform within half a step each way, which below the normal numbers is that of the smallest one."""
    half = torch.finfo(dtype).eps / 2
    return (half * x.abs()).clamp(min=torch.finfo(dtype).smallest_normal * half) ** 2 / 3


@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("d", [64, 128])
def test_small_gradients_in_fp16(d, cap, size):
    """300 tokens over 4096 keys, dO as small as without loss scaling: dS = P (dP - delta) lies among fp16's subnormal numbers.  Its rounding, P's, o's and the results'
    are independent of one another: their variances add up through the sums, and what is measured over some 40000 numbers may be 1.25 times the root of that."""
    dtype, lens, klens, G, scale = torch.float16, [300], [4096], 2, d ** -0.5
    q, k, v, do = inputs(lens, klens, 1, G, d, dtype, 12)
    do = (do.double() * size).to(dtype)
    leaves = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    o, _ = biased_attention(*leaves, cu_of(lens).to(DEV), cu_seqlens_k=cu_of(klens).to(DEV), softcap=cap)
    got = [x.double() for x in torch.autograd.grad(o, leaves, do.to(DEV))]
    q, k, v, do = (x.double().to(DEV) for x in (q, k[:, 0], v[:, 0], do))
    seen, dist = (x.to(DEV) for x in orc.visible(300, 4096))
    sums = [0.0] * 4
    for h in range(G):
        _, lse, dq, dk, dv = orc.one_head(q[:, h], k, v, seen, dist, scale, cap or 0.0, do=do[:, h])[0]
        x = scale * (q[:, h] @ k.T)
        th = torch.tanh(x / cap) if cap else torch.zeros_like(x)
        p = torch.exp2((cap * th if cap else x) / math.log(2.0) - lse[:, None]).masked_fill(~seen, 0.0)
        inner = p * (1 - th * th)
        out = p @ v
        ds = inner * (do[:, h] @ v.T - (out * do[:, h]).sum(1, keepdim=True))
        of_o = spread(p, dtype) * seen @ v ** 2 + spread(out, dtype)
        of_delta = (of_o * do[:, h] ** 2).sum(1, keepdim=True)
        of_ds = spread(ds, dtype) * seen
        of_dq = scale ** 2 * (of_ds @ k ** 2 + of_delta * (inner @ k) ** 2) + spread(dq, dtype)
        assert float((got[0][:, h] - dq).square().mean().sqrt()) <= 1.25 * float(of_dq.mean().sqrt()), f"dq of head {h}"
        sums = [a + b for a, b in zip(sums, (dk, dv, scale ** 2 * (of_ds.T @ q[:, h] ** 2 + (inner ** 2).T @ (of_delta * q[:, h] ** 2)),
                                             (spread(p, dtype) * seen).T @ do[:, h] ** 2))]
    for name, x, ref, of in zip(("dk", "dv"), got[1:], sums[:2], sums[2:]):
        assert float((x[:, 0] - ref).square().mean().sqrt()) <= 1.25 * float((of + spread(ref, dtype)).mean().sqrt()), name


@pytest.mark.parametrize("how", [{}, {"docs": True}, {"window": 40}, {"prefix": [60, 3]}])
@pytest.mark.parametrize("lens,klens", [([100, 30], [300, 90]), ([7, 2], [3000, 2100])])
def test_keys_in_front_of_the_first_sequence(lens, klens, how):
    """cu_seqlens_k as a part of a longer one: the rows in front of it, of NaN, belong to nobody, and their gradients are 0."""
    front, Hk, G, d = 333, 1, 2, 128
    q, k, v, do = inputs(lens, klens, Hk, G, d, BF16, 3)
    ids = torch.div(torch.arange(sum(klens), dtype=torch.int32), 50, rounding_mode="floor").int() if "docs" in how else None
    prefix = torch.tensor(how["prefix"], dtype=torch.int32) if "prefix" in how else None
    ref, off = orc.packed(q, k, v, cu_of(lens), cu_of(klens), d ** -0.5, 20.0, None, how.get("window"), ids, prefix, do, BF16)
    ahead = lambda x, fill: torch.cat([torch.full((front, *x.shape[1:]), fill, dtype=x.dtype), x]).to(DEV)  # noqa: E731
    dirt = [torch.full((front + sum(klens), Hk, d), math.nan, dtype=BF16, device=DEV) for _ in range(4)]
    del dirt                                # (memory for the gradients that does not happen to hold zeros)
    leaves = [x.requires_grad_() for x in (q.to(DEV), ahead(k, math.nan), ahead(v, math.nan))]
    o, lse = biased_attention(*leaves, cu_of(lens).to(DEV), cu_seqlens_k=(cu_of(klens) + front).to(DEV), softcap=20.0, window_size=how.get("window"),
                              doc_ids=None if ids is None else ahead(ids, 0), prefix_lens=None if prefix is None else prefix.to(DEV))
    near(o.detach(), ref[0], off[0], "o")
    near_lse(lse, ref[1])
    dq, dk, dv = torch.autograd.grad(o, leaves, do.to(DEV))
    near(dq, ref[2], off[1], "dq")
    for name, got, r, e in (("dk", dk, ref[3], off[2]), ("dv", dv, ref[4], off[3])):
        near(got[front:], r, e, name)
        assert bool((got[:front] == 0).all()), name


def test_second_derivatives_are_refused():
    """create_graph works for the gradients themselves; what depends on them in turn is refused instead of being left out."""
    lens = [90]
    q, k, v, do = (x.to(DEV) for x in inputs(lens, lens, 1, 2, 64, BF16, 1))
    leaves = [x.requires_grad_() for x in (q, k, v)]

    def first(**how):
        o, _ = biased_attention(*leaves, cu_of(lens).to(DEV), softcap=5.0)
        return torch.autograd.grad(o, leaves, do, **how)

    want, got = first(), first(create_graph=True)
    assert all(torch.equal(a, b.detach()) for a, b in zip(want, got))
    for i in range(3):
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(got[i].float().square().sum() + sum(x.float().sum() for x in leaves), leaves, retain_graph=True)
    torch.autograd.grad(first(retain_graph=True)[0].float().sum() + leaves[0].float().sum(), leaves[0])


def test_backward_without_tokens_writes_dk_and_dv():
    """Through the C ABI: keys that no token is there to see."""
    from fsa import _lib

    cu = torch.zeros(2, dtype=torch.int32, device=DEV)
    dk, dv = (torch.full((50, 2, 64), math.nan, dtype=BF16, device=DEV) for _ in range(2))
    none, p = None, _lib.ptr
    args = [none] * 6 + [p(cu), p(cu)] + [none] * 3 + [0, 50, 1, 4, 2, 64, _lib.DTYPE_CODE[BF16], 256, 64, 128, 128, 256, 64, 0.1, 0.0, -1, none, p(dk), p(dv)]
    args += [none, 0, none, 0, _lib.current_stream(torch.device(DEV))]
    assert _lib.lib().fsa_biased_attn_bwd(*args) == 0
    assert bool((dk == 0).all()) and bool((dv == 0).all())


@pytest.mark.parametrize("G", [3, 7, 11, 31])
@pytest.mark.parametrize("d", [64, 128])
def test_the_same_bits_whatever_a_kernel_before_left(G, d):
    """Groups whose heads do not fill a tile's 128 rows: what stands in the other rows' shared memory, zeros or numbers far above every cap, changes no bit."""
    lens, P = [150, 33], 300
    q, k, v, do = (x.to(DEV) for x in inputs(lens, lens, 2, G, d, BF16, G))
    cu, sl = cu_of(lens).to(DEV), slopes_of(2 * G).to(DEV)
    big = [torch.ones(9000, h, d, dtype=BF16, device=DEV) for h in (4, 1, 1, 4)]
    n, pre = i32([2, 5, 1, 9]), [k[:P], v[:P], i32([0, 150, 183]), i32([0, 3, 4])]
    k2, v2 = (x.repeat(2, 1, 1) for x in (k, v))
    r0 = i32([0, 10, 20, 30])

    def fill(value):
        """Every SM's shared memory, by the same kernels on tiles that are full."""
        leaves = [(x * value).requires_grad_() for x in big[:3]]
        o, _ = biased_attention(*leaves, i32([0, 9000]), softcap=5.0)
        torch.autograd.grad(o, leaves, big[3] * value)

    def run(cap, alibi):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        o, lse = biased_attention(*leaves, cu, softcap=cap, alibi_slopes=sl if alibi else None)
        return [o.detach(), lse, *torch.autograd.grad(o, leaves, do),
                *shared_prefix_decode_attention(q[:4], k2, v2, n, r0, *pre, max_len=9, softcap=cap, alibi_slopes=sl if alibi else None)]

    for cap, alibi in SCORES_OF:
        fill(0.0)
        want = run(cap, alibi)
        for value in (1e3, -1e3):
            fill(value)
            assert all(torch.equal(a, b) for a, b in zip(want, run(cap, alibi))), (cap, alibi, value)


@pytest.mark.parametrize("G,d", [(2, 128), (3, 64), (1, 64)])
@pytest.mark.parametrize("how", [{}, {"docs": True}, {"window": 70}])
def test_the_same_bits_whatever_nobodys_rows_hold(G, d, how):
    """Rows in front of, behind and (as padding) within the sequences: zeros, numbers far above every cap, NaN.  No bit of the others' results changes."""
    lens, klens, front, behind = [150, 90, 33], [300, 90, 200], 77, 50
    q, k, v, do = inputs(lens, klens, 2, G, d, BF16, 20 + G)
    ids = None
    if "docs" in how:
        ids = torch.cat([torch.full((n,), i, dtype=torch.int32) for n, i in ((200, 1), (70, -1), (90, 2), (60, 3), (100, -2), (70, 4))])
    sl, cu, cuk = slopes_of(2 * G).to(DEV), cu_of(lens).to(DEV), (cu_of(klens) + front).to(DEV)

    def run(value, cap, alibi):
        def pad(x, a, b):
            y = torch.full((a + x.shape[0] + b, *x.shape[1:]), value, dtype=x.dtype)
            y[a : a + x.shape[0]] = x
            return y

        kk, vv, qq, dd = pad(k, front, behind), pad(v, front, behind), pad(q, 0, behind), pad(do, 0, behind)
        if ids is not None:
            nobody = torch.nonzero(ids < 0)[:, 0]
            kk[front + nobody], vv[front + nobody] = value, value
            at = torch.cat([torch.arange(c, c + n) for c, n in ((150, 150), (300, 90), (557, 33))])       # keys at which the tokens stand
            qq[: len(at)][ids[at] < 0], dd[: len(at)][ids[at] < 0] = value, value
        leaves = [x.to(DEV).requires_grad_() for x in (qq, kk, vv)]
        docs = None if ids is None else torch.cat([torch.zeros(front, dtype=torch.int32), ids, torch.zeros(behind, dtype=torch.int32)]).to(DEV)
        o, lse = biased_attention(*leaves, cu, cu_seqlens_k=cuk, softcap=cap, alibi_slopes=sl if alibi else None, doc_ids=docs, window_size=how.get("window"))
        return [o.detach(), lse, *torch.autograd.grad(o, leaves, dd.to(DEV))]

    for cap, alibi in SCORES_OF:
        want = run(0.0, cap, alibi)
        for value in (1e3, -1e4, math.nan):
            assert all(torch.equal(a, b) for a, b in zip(want, run(value, cap, alibi))), (cap, alibi, value)


@pytest.mark.parametrize("how", [{}, {"docs": True}, {"window": 50}, {"prefix": True}])
def test_a_captured_step_with_other_lengths(how):
    """Lengths, documents and prefixes are read on the device: a captured step is replayed with others, and gives what an eager one gives for them."""
    n, B = 700, 3
    q, k, v, do = (x.to(DEV) for x in inputs([n], [n], 2, 2, 64, BF16, 30))
    cu, cuk, ids, prefix = i32([0, 300, 500, n]), i32([0, 300, 500, n]), i32([t // 90 for t in range(n)]), i32([10, 0, 50])
    leaves = [x.requires_grad_() for x in (q, k, v)]

    def step():
        o, lse = biased_attention(*leaves, cu, cu_seqlens_k=cuk, softcap=30.0, doc_ids=ids if "docs" in how else None, window_size=how.get("window"),
                                  prefix_lens=prefix if "prefix" in how else None)
        return [o.detach(), lse, *torch.autograd.grad(o, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for lens, klens in (([1, 0, 600], [500, 100, 100]), ([0, 0, 0], [0, 0, 0]), ([233, 233, 234], [233, 233, 234]), ([700, 0, 0], [100, 300, 200])):
        assert len(lens) == B
        cu.copy_(cu_of(lens))
        cuk.copy_(cu_of(klens))
        ids.copy_(torch.div(torch.arange(n, dtype=torch.int32), 7 + lens[0] % 50, rounding_mode="floor").int() % 5 - 1)
        prefix.copy_(torch.tensor([lens[0] // 2, -4, 1000], dtype=torch.int32))
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), (lens, klens)


def test_memory_that_calls_find_changes_no_bit():
    """Workspaces and results lie where something else was: all bits set, or zeros."""
    lens, klens = [400, 1, 90, 33], [900, 300, 90, 200]
    q, k, v, do = (x.to(DEV) for x in inputs(lens, klens, 1, 4, 128, BF16, 31))
    cu, cuk, ids = cu_of(lens).to(DEV), cu_of(klens).to(DEV), i32([t // 60 for t in range(sum(klens))])
    n, r0, pre = i32([5, 0, 300, 1]), i32([0, 10, 400, 800]), [k[:260], v[:260], i32([0, 200, 260]), i32([1, 2, 3])]

    def run():
        out = []
        for how in ({}, {"doc_ids": ids}, {"window_size": 100}):
            leaves = [x.detach().requires_grad_() for x in (q, k, v)]
            o, lse = biased_attention(*leaves, cu, cu_seqlens_k=cuk, softcap=30.0, **how)
            out += [o.detach(), lse, *torch.autograd.grad(o, leaves, do)]
        one = [x.detach().requires_grad_() for x in (q[:400, :1], k, v)]            # few items: o and dQ cut along the keys
        o, lse = biased_attention(*one, i32([0, 400]), cu_seqlens_k=i32([0, sum(klens)]), softcap=30.0)
        out += [o.detach(), lse, *torch.autograd.grad(o, one, do[:400, :1])]
        out += biased_decode_attention(q[:4], k, v, n, r0, max_len=300)
        return out + list(shared_prefix_decode_attention(q[:4], k, v, n, r0, *pre, max_len=300))

    want = run()
    for byte in (0, 255):
        for size in [1 << i for i in range(9, 27)] * 3:
            torch.full((size,), byte, dtype=torch.uint8, device=DEV)
        held = [torch.full((size,), byte, dtype=torch.uint8, device=DEV) for size in [1 << i for i in range(9, 26)] * 4]
        del held
        assert all(torch.equal(a, b) for a, b in zip(want, run())), byte
