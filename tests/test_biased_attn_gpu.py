"""Attention with changed scores and masks against its definition in 64 bits.

Allowances (derived, not fitted): the kernels round P and dS to the 16-bit type before they are multiplied, the results once, and take
sum(o dO) from the rounded o; each rounding is off by at most half a step, finfo.eps / 2 of the value, or of the smallest normal number below
it.  ``biased_attn_oracle`` carries these through the sums.  What is done in 32 bits comes on top: sums of up to 4096 terms, scores of up
to 64 whose error of 2^-20 (tanh: 6e-7 of it) becomes 6e-5 of a probability: SLACK of the whole, and 2^-20 of the largest value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fsa.ops import biased_attention
from oracle import biased_attn_oracle as orc

DEV = "cuda:0"
SLACK = 1.05
BF16, FP16 = torch.bfloat16, torch.float16


def cu_of(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)


def slopes_of(Hq):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / Hq) for i in range(Hq)])


def inputs(lens, klens, Hk, G, d, dtype, seed, qsize=2.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda n, h, s=1.0: (torch.randn(n, h, d, generator=g) * s).to(dtype)  # noqa: E731
    N, Nk = sum(lens), sum(klens)
    return mk(N, Hk * G, qsize), mk(Nk, Hk), mk(Nk, Hk), mk(N, Hk * G)


def near(got, ref, off, name):
    err = (got.double().cpu() - ref).abs()
    room = SLACK * off + 2.0 ** -20 * float(ref.abs().max() if ref.numel() else 0)
    assert not torch.isnan(err).any(), f"{name}: NaN"
    assert bool((err <= room).all()), f"{name}: {float((err - room).max()):.3e} over the allowance, error {float(err.max()):.3e}"


def near_lse(got, ref):
    """32-bit scores of up to 2^6.5 log2 units: 2^-17 each way, and the sum's 2^-20."""
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got.cpu()), fin) and bool((got.cpu()[~fin] == -math.inf).all())
    if fin.any():
        assert float((got.double().cpu() - ref)[fin].abs().max()) <= 2.0 ** -16 * max(1.0, float(ref[fin].abs().max()) / 16)


def check(q, k, v, do, lens, klens, cap=None, slopes=None, window=None, ids=None, prefix=None, scale=None):
    dtype, d = q.dtype, q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    cu, cuk = cu_of(lens), cu_of(klens)
    ref, off = orc.packed(q, k, v, cu, cuk, scale, cap or 0.0, slopes, window, ids, prefix, do, dtype)
    dev = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    qc, kc, vc = (x.detach().to(DEV).requires_grad_() for x in (q, k, v))
    o, lse = biased_attention(qc, kc, vc, cu.to(DEV), cu_seqlens_k=None if lens == klens else cuk.to(DEV), sm_scale=scale, softcap=cap,
                              alibi_slopes=dev(slopes), window_size=window, doc_ids=dev(ids), prefix_lens=dev(prefix))
    assert o.dtype == dtype and lse.dtype == torch.float32 and not lse.requires_grad
    grads = torch.autograd.grad(o, (qc, kc, vc), do.to(DEV))
    near(o.detach(), ref[0], off[0], "o")
    near_lse(lse, ref[1])
    for name, got, r, e in zip(("dq", "dk", "dv"), grads, ref[2:], off[1:]):
        near(got, r, e, name)
    return o, lse, grads


SCORES = {"plain": (None, False), "cap": (20.0, False), "alibi": (None, True), "both": (50.0, True)}


@pytest.mark.parametrize("score", list(SCORES))
@pytest.mark.parametrize("lens,Hk,G,d,dtype", [
    ([300, 45, 212], 2, 2, 128, BF16),
    ([1], 1, 1, 128, BF16),                          # one token
    ([1, 2, 0, 63, 64, 65, 129], 2, 4, 64, FP16),    # around a tile's 64 rows, a sequence without tokens
    ([517], 1, 3, 128, FP16),                        # 40 tokens a tile: 120 of its 128 rows are used
    ([260, 9], 1, 16, 64, BF16),                     # 8 tokens a tile
    ([130], 1, 32, 128, BF16),
    ([33, 70, 5, 128] * 9, 1, 2, 128, BF16),         # 36 sequences: the lookup walks them 32 at a time
    ([1300], 1, 1, 64, BF16),
])
def test_causal(score, lens, Hk, G, d, dtype):
    cap, alibi = SCORES[score]
    q, k, v, do = inputs(lens, lens, Hk, G, d, dtype, sum(lens) + G)
    check(q, k, v, do, lens, lens, cap, slopes_of(Hk * G) if alibi else None)


@pytest.mark.parametrize("score", list(SCORES))
@pytest.mark.parametrize("window", [0, 1, 63, 64, 100, 5000])
def test_window(score, window):
    cap, alibi = SCORES[score]
    lens = [400, 77]
    q, k, v, do = inputs(lens, lens, 2, 2, 128, BF16, window)
    check(q, k, v, do, lens, lens, cap, slopes_of(4) if alibi else None, window=window)


@pytest.mark.parametrize("d,dtype,G", [(128, BF16, 4), (64, FP16, 2)])
@pytest.mark.parametrize("score", list(SCORES))
def test_documents_and_padding(score, d, dtype, G):
    """Documents of one token, across tiles, equal ids apart from one another, padding between and behind: what stands in the padded rows of
    q, k, v and dO is NaN or infinite."""
    cap, alibi = SCORES[score]
    lens = [700, 1, 300, 90]
    pieces = [(64, 0), (1, 1), (1, 2), (200, 0), (34, -1), (300, 5), (100, -7), (1, 3), (150, 4), (150, 6), (90, -1)]
    ids = torch.cat([torch.full((n,), i, dtype=torch.int32) for n, i in pieces])
    assert len(ids) == sum(lens)
    q, k, v, do = inputs(lens, lens, 2, G, d, dtype, 5)
    bad = torch.nonzero(ids < 0)[:, 0]
    for i, x in enumerate((q, k, v, do)):
        x[bad] = math.nan
        x[bad[i::3]] = math.inf if i % 2 else -math.inf
    check(q, k, v, do, lens, lens, cap, slopes_of(2 * G) if alibi else None, ids=ids)


@pytest.mark.parametrize("prefix", [[0, 0, 0], [300, 45, 212], [131, 1, 211], [1000, 64, 0]])
@pytest.mark.parametrize("score", list(SCORES))
def test_prefix(score, prefix):
    """(A prefix longer than its sequence is all of it.)"""
    cap, alibi = SCORES[score]
    lens = [300, 45, 212]
    q, k, v, do = inputs(lens, lens, 2, 2, 128, BF16, sum(prefix))
    check(q, k, v, do, lens, lens, cap, slopes_of(4) if alibi else None, prefix=torch.tensor(prefix, dtype=torch.int32))


@pytest.mark.parametrize("score", list(SCORES))
@pytest.mark.parametrize("lens,klens,how", [
    ([64, 1, 200], [500, 333, 200], {}),
    ([64, 1, 200], [500, 333, 200], {"window": 70}),
    ([7, 130], [7 + 512, 1000], {"docs": True}),
    ([100, 5, 0, 3], [40, 0, 77, 3], {}),             # fewer keys than queries: the first ones see nothing
    ([300, 60], [700, 64], {"prefix": [650, 10]}),
])
def test_chunked_prefill(score, lens, klens, how):
    cap, alibi = SCORES[score]
    q, k, v, do = inputs(lens, klens, 1, 4, 128, BF16, sum(klens))
    ids = None
    if how.get("docs"):
        g = torch.Generator().manual_seed(1)
        ids = torch.cumsum((torch.rand(sum(klens), generator=g) < 0.01).int(), 0).to(torch.int32)
    prefix = torch.tensor(how["prefix"], dtype=torch.int32) if "prefix" in how else None
    check(q, k, v, do, lens, klens, cap, slopes_of(4) if alibi else None, window=how.get("window"), ids=ids, prefix=prefix)


@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, FP16)])
def test_saturated_cap(d, dtype):
    """Scores far above the cap, on both sides of zero: both forms of the tanh, its derivative down to 0."""
    lens = [150, 201]
    q, k, v, do = inputs(lens, lens, 2, 2, d, dtype, 3, qsize=8.0)
    q[100:200] *= 6
    check(q, k, v, do, lens, lens, cap=5.0)


def test_documents_of_thousands_of_tokens():
    """The search for a document's beginning goes back further than its step of 512 ids."""
    lens = [2600]
    ids = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate((700, 1800, 100))])
    q, k, v, do = inputs(lens, lens, 1, 2, 64, BF16, 8)
    check(q, k, v, do, lens, lens, cap=30.0, ids=ids)


def test_strided_rows_and_broadcast_gradients():
    """q, k, v as views of a fused projection, transposed heads, and the expanded gradient of a sum."""
    lens, Hk, G, d = [200, 31], 2, 2, 128
    N, Hq = sum(lens), Hk * G
    g = torch.Generator().manual_seed(4)
    fused = torch.randn(N, (Hq + 2 * Hk) * d, generator=g).to(BF16)
    q, k, v = fused[:, : Hq * d].view(N, Hq, d), fused[:, Hq * d : (Hq + Hk) * d].view(N, Hk, d), fused[:, (Hq + Hk) * d :].view(N, Hk, d)
    cu = cu_of(lens)
    ref, off = orc.packed(q, k, v, cu, cu, d ** -0.5, 30.0, slopes_of(Hq), do=torch.ones(N, Hq, d), dtype=BF16)
    f = fused.to(DEV).requires_grad_()
    fq, fk, fv = f[:, : Hq * d].view(N, Hq, d), f[:, Hq * d : (Hq + Hk) * d].view(N, Hk, d), f[:, (Hq + Hk) * d :].view(N, Hk, d)
    o, _ = biased_attention(fq, fk, fv, cu.to(DEV), softcap=30.0, alibi_slopes=slopes_of(Hq).to(DEV))
    near(o.detach(), ref[0], off[0], "o")
    o.sum().backward()
    want, room = torch.cat([x.flatten(1) for x in ref[2:]], 1), torch.cat([x.flatten(1) for x in off[1:]], 1)
    near(f.grad, want, room, "gradient of the fused projection")
    ht = q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)           # heads outside
    o2, _ = biased_attention(ht, k.to(DEV), v.to(DEV), cu.to(DEV), softcap=30.0, alibi_slopes=slopes_of(Hq).to(DEV))
    assert torch.equal(o2, o.detach())


def test_rows_behind_the_last_sequence():
    """A buffer with room: rows behind cu_seqlens[-1] hold NaN, o is 0 and lse -inf there, gradients are 0."""
    lens, room, Hk, G, d = [130, 70], 333, 2, 2, 128
    q, k, v, do = inputs(lens, lens, Hk, G, d, BF16, 6)
    pad = lambda x: torch.cat([x, torch.full((room, *x.shape[1:]), math.nan, dtype=x.dtype)]).to(DEV)  # noqa: E731
    qc, kc, vc = (pad(x).requires_grad_() for x in (q, k, v))
    cu = cu_of(lens)
    ref, off = orc.packed(q, k, v, cu, cu, d ** -0.5, 50.0, do=do, dtype=BF16)
    o, lse = biased_attention(qc, kc, vc, cu.to(DEV), softcap=50.0)
    n = sum(lens)
    near(o.detach()[:n], ref[0], off[0], "o")
    assert bool((o[n:] == 0).all()) and bool((lse[:, n:] == -math.inf).all())
    for name, got, r, e in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (qc, kc, vc), pad(do)), ref[2:], off[1:]):
        near(got[:n], r, e, name)
        assert bool((got[n:] == 0).all()), name


def test_empty_inputs():
    z = lambda n, h: torch.zeros(n, h, 64, dtype=BF16, device=DEV, requires_grad=True)  # noqa: E731
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    o, lse = biased_attention(z(0, 4), z(0, 2), z(0, 2), i32(0, 0))
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
    q, k = z(5, 4), z(0, 2)
    o, lse = biased_attention(q, k, k, i32(0, 5), cu_seqlens_k=i32(0, 0), softcap=3.0)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    assert all(bool((g == 0).all()) for g in torch.autograd.grad(o.sum(), (q, k)))


def test_the_same_bits_from_run_to_run_and_from_a_graph():
    lens, Hk, G, d = [900, 333], 2, 4, 128
    q, k, v, do = (x.to(DEV) for x in inputs(lens, lens, Hk, G, d, BF16, 7))
    cu, sl = cu_of(lens).to(DEV), slopes_of(Hk * G).to(DEV)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]

    def step():
        o, lse = biased_attention(*leaves, cu, softcap=50.0, alibi_slopes=sl)
        return [o.detach(), lse, *torch.autograd.grad(o, leaves, do)]

    first, again = step(), step()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        leaves[0].copy_(q * 0.5)
    graph.replay()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(held, want)) and not torch.equal(held[0], first[0])


def test_two_streams_at_once():
    lens = [700, 200]
    cu = cu_of(lens).to(DEV)
    sets = [[x.to(DEV) for x in inputs(lens, lens, 2, 2, 128, BF16, s)[:3]] for s in (1, 2)]
    want = [biased_attention(*x, cu, softcap=20.0) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for st, x in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(biased_attention(*x, cu, softcap=20.0))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
