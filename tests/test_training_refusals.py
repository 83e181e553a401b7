"""What the training operators refuse, on the host (CPU): the checks come before
the one for CUDA tensors."""

import pytest
import torch
from torch.autograd import forward_ad

import llm_hgemm
from llm_hgemm import capi, train_capi, training


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


ADDRESS = 1 << 20   # aligned, never read


@pytest.mark.parametrize("field, off", [("target", 4), ("lse", 2), ("loss", 2)])
def test_c_abi_refuses_misaligned_loss_arrays(field, off):
    a = train_capi.LossForward(train_capi.Common(), *[ADDRESS] * 6, 1 << 30, 4, 16, 100, 16, -100, 0, 0)
    setattr(a, field, ADDRESS + off)
    assert train_capi.run("loss_forward", a) == capi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("field, off", [("target", 4), ("lse", 2), ("dloss", 2)])
def test_c_abi_refuses_misaligned_loss_gradient_arrays(field, off):
    a = train_capi.LossBackward(train_capi.Common(), *[ADDRESS] * 8, 1 << 30, 4, 16, 100, 16, -100, 0, 0, 0)
    setattr(a, field, ADDRESS + off)
    assert train_capi.run("loss_backward", a) == capi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("field", ["g", "out"])
@pytest.mark.parametrize("rows", [100, 200])
def test_c_abi_refuses_misaligned_updates(field, rows):
    a = train_capi.Orthogonalize(train_capi.Common(), *[ADDRESS] * 3, 1 << 30, 1, rows, 300, 300, 0, 5, 0,
                                 *training.NEWTON_SCHULZ, 0.0, 1e-7)
    setattr(a, field, ADDRESS + 1)
    assert train_capi.run("orthogonalize", a) == capi.ERR_INVALID_ARGUMENT


def test_c_abi_refuses_a_misaligned_status_word():
    a = train_capi.FfnForward(train_capi.Common(status=ADDRESS + 2), *[ADDRESS] * 6, None, None, None, 0,
                              16, 64, 128, 64, 64)
    assert train_capi.run("ffn_forward", a) == capi.ERR_INVALID_ARGUMENT
