"""What the decode operators with changed scores refuse (no GPU needed), and how their work is cut."""
import math
from ctypes import byref, c_int64

import pytest
import torch

from fsa import _lib
from fsa_preview.ops import biased_decode_attention, shared_prefix_decode_attention

BF16 = torch.bfloat16


def _args(B=3, rows=20, Hq=4, Hk=2, d=64, dtype=BF16):
    i = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    return [torch.zeros(B, Hq, d, dtype=dtype), torch.zeros(rows, Hk, d, dtype=dtype), torch.zeros(rows, Hk, d, dtype=dtype), i(B), i(B)]


def _prefix(P=7, Hk=2, d=64, n=1):
    i = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    return [torch.zeros(P, Hk, d, dtype=BF16), torch.zeros(P, Hk, d, dtype=BF16), i(n + 1), i(n + 1)]


@pytest.mark.parametrize("change,error", [
    (dict(dtype=torch.float32), TypeError),
    (dict(Hq=3), ValueError),
    (dict(d=256), ValueError),
    (dict(Hq=66), ValueError),
])
def test_refuses_shapes(change, error):
    with pytest.raises(error):
        biased_decode_attention(*_args(**change), max_len=5)
    with pytest.raises(error):
        shared_prefix_decode_attention(*_args(**change), *_prefix(), max_len=5)


@pytest.mark.parametrize("how,error", [
    (dict(softcap=-1.0), ValueError),
    (dict(softcap=math.nan), ValueError),
    (dict(sm_scale=-2.0), ValueError),
    (dict(window_size=-1), ValueError),
    (dict(alibi_slopes=torch.zeros(3)), ValueError),
    (dict(alibi_slopes=torch.zeros(4, dtype=BF16)), TypeError),
    (dict(max_len=-1), ValueError),
    (dict(), ValueError),                    # no CUDA tensors
])
def test_refuses_arguments(how, error):
    with pytest.raises(error):
        biased_decode_attention(*_args(), **{"max_len": 5, **how})
    with pytest.raises(error):
        shared_prefix_decode_attention(*_args(), *_prefix(), **{"max_len": 5, **how})


def test_refuses_lengths():
    a = _args()
    with pytest.raises(TypeError):
        biased_decode_attention(*a[:3], a[3].long(), a[4], max_len=5)
    with pytest.raises(ValueError):
        biased_decode_attention(*a[:4], a[4][:2], max_len=5)


@pytest.mark.parametrize("at,other", [(0, _prefix(Hk=1)[0]), (0, _prefix(P=6)[0]), (1, _prefix(d=128)[1]), (2, torch.zeros(1, dtype=torch.int32)),
                                      (3, torch.zeros(3, dtype=torch.int32)), (2, torch.zeros(2, dtype=torch.int64))])
def test_refuses_prefixes(at, other):
    p = _prefix()
    p[at] = other
    with pytest.raises((ValueError, TypeError)):
        shared_prefix_decode_attention(*_args(), *p, max_len=5)


def _bytes(B, Hq, Hk, D, groups, max_len, max_shared, window=-1):
    n = c_int64(0)
    assert _lib.lib().fsa_biased_decode_bytes(B, Hq, Hk, D, groups, max_len, max_shared, window, byref(n)) == 0
    return n.value


def test_workspace_holds_the_partials_and_no_more_than_it_has_to():
    per = lambda B, Hq, D, P: B * Hq * P * (D * 4 + 8)  # noqa: E731
    assert _bytes(1, 32, 8, 128, 0, 1, 0) >= per(1, 32, 128, 1)
    assert _bytes(64, 32, 8, 128, 0, 16384, 0) <= per(64, 32, 128, 16) + 512              # chunks of 1024 rows
    assert _bytes(64, 32, 8, 128, 0, 16384, 0, window=511) <= per(64, 32, 128, 8) + 512    # no more than the window is cut
    # a prefix of 32768 rows, 64 sequences in two tiles a kv head: some 19 chunks
    assert per(64, 32, 128, 20) <= _bytes(64, 32, 8, 128, 1, 1024, 32768) <= per(64, 32, 128, 36) + 512
    L, n = _lib.lib(), c_int64(0)
    assert L.fsa_biased_decode_bytes(1, 3, 2, 128, 0, 1, 0, -1, byref(n)) == _lib.FSA_ERR_BAD_ARG
    assert L.fsa_biased_decode_bytes(1, 4, 2, 256, 0, 1, 0, -1, byref(n)) == _lib.FSA_ERR_UNSUPPORTED
    assert L.fsa_biased_decode_bytes(1, 66, 2, 128, 0, 1, 0, -1, byref(n)) == _lib.FSA_ERR_UNSUPPORTED
    assert L.fsa_biased_attn_bwd_bytes(10, 10, 0, 4, 2, 128, -1, byref(n)) == _lib.FSA_ERR_BAD_ARG
    assert L.fsa_biased_attn_bwd_bytes(1 << 25, 10, 1, 4, 2, 128, -1, byref(n)) == _lib.FSA_ERR_UNSUPPORTED
