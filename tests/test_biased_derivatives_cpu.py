"""Derivatives that the attention with changed scores does not have are refused, not dropped (no GPU needed)."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from fsa.ops import biased_attention
from fsa_preview.ops import biased_decode_attention, shared_prefix_decode_attention

BF16 = torch.bfloat16


@pytest.mark.parametrize("at", [0, 1, 2])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode(at, grad):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    x = [torch.zeros(6, h, 64, dtype=BF16) for h in (4, 2, 2)]
    with fwAD.dual_level():
        x[at] = fwAD.make_dual(x[at].requires_grad_(grad), torch.ones_like(x[at]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            biased_attention(*x, i32(0, 6))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            biased_decode_attention(x[0], x[1], x[2], i32(*[1] * 6), i32(*range(6)), max_len=1)
        plain = [torch.zeros(6, h, 64, dtype=BF16) for h in (4, 2, 2)]
        if at:
            pre = [torch.zeros(6, 2, 64, dtype=BF16) for _ in range(2)]
            pre[at - 1] = x[at]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                shared_prefix_decode_attention(*plain, i32(*[1] * 6), i32(*range(6)), *pre, i32(0, 6), i32(0, 6), max_len=1)
        # (other tensors of a dual level may come)
        with pytest.raises(ValueError, match="CUDA"):
            biased_attention(*plain, i32(0, 6))


def test_forward_mode_of_the_slopes():
    x = [torch.zeros(6, h, 64, dtype=BF16) for h in (4, 2, 2)]
    with fwAD.dual_level():
        slopes = fwAD.make_dual(torch.zeros(4), torch.ones(4))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            biased_attention(*x, torch.tensor([0, 6], dtype=torch.int32), alibi_slopes=slopes)
