"""What the training operators refuse, on the host (CPU): the checks come before
the one for CUDA tensors."""

import pytest
import torch
from torch.autograd import forward_ad

import llm_hgemm


@pytest.mark.parametrize("which", range(4))
def test_forward_mode_of_the_ffn_is_refused(which):
    shapes = ((4, 8), (16, 8), (16, 8), (8, 16))
    args = [torch.ones(s, dtype=torch.float16) for s in shapes]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="gated_ffn has no forward-mode derivative"):
            llm_hgemm.gated_ffn(*args)


@pytest.mark.parametrize("which", range(2))
def test_forward_mode_of_the_loss_is_refused(which):
    args = [torch.ones(4, 8, dtype=torch.float16), torch.ones(16, 8, dtype=torch.float16)]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="linear_cross_entropy has no forward-mode derivative"):
            llm_hgemm.linear_cross_entropy(*args, torch.zeros(4, dtype=torch.int64))
