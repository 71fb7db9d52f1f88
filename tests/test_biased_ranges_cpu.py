"""Ends of the arguments' ranges that the attention with changed scores refuses, without a GPU."""
import ctypes

import pytest
import torch

from fsa.ops import biased_attention
from fsa_preview.ops import biased_decode_attention
from fsa._lib import FSA_ERR_UNSUPPORTED, lib


@pytest.mark.parametrize("how", [
    {"softcap": 1e-31}, {"softcap": 1e31}, {"softcap": 1e-20, "sm_scale": 1e15}, {"softcap": 1e25, "sm_scale": 1e-10},
    {"softcap": float("nan")}, {"softcap": float("inf")}, {"sm_scale": float("inf")},
])
def test_caps_whose_numbers_leave_32_bits(how):
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    n = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="softcap|sm_scale"):
        biased_attention(x, x, x, n, **how)
    with pytest.raises(ValueError, match="softcap|sm_scale"):
        biased_decode_attention(x, x, x, torch.ones(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), max_len=4, **how)


@pytest.mark.parametrize("max_len,max_shared", [(1 << 30, 0), (1 << 62, 0), (1, 1 << 40)])
def test_lengths_that_no_cache_has(max_len, max_shared):
    out = ctypes.c_int64(-7)
    assert lib().fsa_biased_decode_bytes(4, 8, 2, 64, 2, max_len, max_shared, -1, ctypes.byref(out)) == FSA_ERR_UNSUPPORTED
    assert out.value == -7


@pytest.mark.parametrize("scale", [1e39, 3e38, 1e-50, 1e-40])
def test_scales_that_leave_32_bits(scale):
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="sm_scale"):
        biased_attention(x, x, x, torch.tensor([0, 4], dtype=torch.int32), sm_scale=scale)
    with pytest.raises(ValueError, match="sm_scale"):
        biased_decode_attention(x, x, x, torch.ones(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), max_len=4, sm_scale=scale)


@pytest.mark.parametrize("batch,kv_heads,fits", [(1 << 20, 8, True), (1 << 24, 64, False), (1 << 24, 256, False), (1 << 23, 127, True)])
def test_more_places_than_a_grid_has(batch, kv_heads, fits):
    """Sequences without tokens take a place in the list of tiles too: their number times the kv heads stays in 32 bits."""
    out = ctypes.c_int64(-7)
    want = 0 if fits else FSA_ERR_UNSUPPORTED
    for size in (lib().fsa_biased_attn_fwd_bytes, lib().fsa_biased_attn_bwd_bytes):
        assert size(5, 1000, batch, kv_heads, kv_heads, 64, -1, ctypes.byref(out)) == want
    assert lib().fsa_biased_decode_bytes(4, kv_heads, kv_heads, 64, batch, 100, 100, -1, ctypes.byref(out)) == want
