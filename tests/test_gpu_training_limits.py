"""Training operators where a call meets a limit of its kernels (GPU)."""

import ctypes

import pytest
import torch

import llm_hgemm
from llm_hgemm import _C, capi, train_capi, training
from tests import training_reference as ref
from tests.gpu_helpers import require_cuda
from tests.test_gpu_training import DTYPES, IDS, ffn_inputs, ffn_through_c, loss_inputs, loss_through_c, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    require_cuda()


@pytest.mark.parametrize("tokens, vocab, piece, tile", [
    (2049, 8256, 8192, 128), (3841, 4672, 4608, 256 | train_capi.TILE_PAIR), (8192, 9108, 0, 0),
], ids=["single", "pair", "chosen"])
def test_loss_short_last_piece_of_many_tile_rows(tokens, vocab, piece, tile):
    """At least 16 rows of tiles, where the raster's groups of rows depend on the
    sum's length: a last piece short enough for taller groups still adds each tile
    of dx to its own."""
    x, w, t = loss_inputs(tokens, 520, vocab, torch.bfloat16)
    dl = torch.tensor([64.0], device="cuda")
    want = ref.loss(x, w, t, "sum", -100, dl)
    got = loss_through_c(x, w, t, dl, tile, piece, train_capi.LOSS_SUM)
    for g, v in zip((got[0][0], got[1], got[2]), want):
        within(g, v)


@pytest.mark.parametrize("wanted, piece", [("both", 0), ("both", 4096), ("x", 0), ("weight", 0)])
@pytest.mark.parametrize("dtype, sizes", [
    (torch.float16, [2e4, 1e-3, 1.0, -3e-3, 0.0, 5e-5]),
    (torch.bfloat16, [1e20, 1e-20, 1.0, -3e-22, 0.0, 5e4]),
    (torch.bfloat16, [1e-35, -3e-35, 2e-36, 1e-35, 0.0, 1e-37]),
    (torch.bfloat16, [3.4e38, -3.4e38, 1.0, 1e30, 0.0, 1e8]),
], ids=["fp16", "bf16", "bf16 tiny", "bf16 huge"])
def test_loss_gradients_of_small_and_large_rows(dtype, sizes, wanted, piece):
    """Every row of dx is as good as if it were the only one, whatever the other
    rows' incoming gradients. The weights have a mean, so that the probabilities'
    part of a row (each of them 1/20011) is as large as its target's."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    w = (0.5 + 0.05 * torch.randn(20011, 64, generator=gen, device="cuda")).to(dtype)
    x = (0.05 * torch.randn(6, 64, generator=gen, device="cuda")).to(dtype)
    t = torch.arange(6, device="cuda") * 3000
    dl = torch.tensor(sizes, device="cuda")
    if piece:
        _, dx, dw = loss_through_c(x, w, t, dl, piece=piece, reduction=train_capi.LOSS_NONE)
    else:
        leaves = [v.requires_grad_() for v, name in ((x, "x"), (w, "weight")) if wanted in ("both", name)]
        grads = list(torch.autograd.grad(llm_hgemm.linear_cross_entropy(x, w, t, reduction="none"), leaves, dl))
        dx = grads.pop(0) if wanted != "weight" else None
        dw = grads.pop(0) if wanted != "x" else None
    if dx is not None:
        for i in range(6):
            within(dx[i:i + 1], ref.loss(x[i:i + 1], w, t[i:i + 1], "none", -100, dl[i:i + 1])[1])
    if dw is not None:
        within(dw, ref.loss(x, w, t, "none", -100, dl)[2])


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_loss_infinite_gradients_stay_in_their_rows(dtype, bad):
    """An incoming gradient that is infinite or NaN reaches its own row of dx, or
    all rows with a target where there is one for all, and no ignored row."""
    x, w, t = loss_inputs(40, 64, 500, dtype)
    t[3], t[7] = -100, 5
    keep = t != -100
    x.requires_grad_()
    dl = torch.linspace(-2.0, 3.0, 40, device="cuda")
    want = ref.loss(x, w, t, "none", -100, dl)[1]
    dl[7] = bad
    (dx,) = torch.autograd.grad(llm_hgemm.linear_cross_entropy(x, w, t, reduction="none"), x, dl)
    others = torch.arange(40, device="cuda") != 7
    assert not dx[7].isfinite().any()
    within(dx[others], (want[0][others], want[1][others]))
    for reduction in ("sum", "mean"):
        value = llm_hgemm.linear_cross_entropy(x, w, t, reduction=reduction)
        (dx,) = torch.autograd.grad(value, x, torch.tensor(bad, device="cuda"))
        assert not dx[keep].isfinite().any() and not dx[~keep].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("size", [(40, 64, 500), (333, 37, 1001), (1500, 264, 700)], ids=str)
def test_loss_ignored_rows_may_hold_anything(size, reduction, dtype):
    """Infinity and NaN in ignored rows reach neither the loss, dx nor dW."""
    x, w, t = loss_inputs(*size, dtype)
    t[3] = t[9] = t[-1] = -100
    keep = t != -100
    gen = torch.Generator(device="cuda").manual_seed(8)
    dl = (torch.rand(size[0], generator=gen, device="cuda") if reduction == "none" else torch.ones((), device="cuda"))
    want = ref.loss(x[keep], w, t[keep], reduction, -100, dl[keep] if reduction == "none" else dl)
    poisoned = x.clone()
    poisoned[~keep] = float("inf")
    poisoned[3] = float("nan")
    poisoned[9, 1:] = x[9, 1:]
    poisoned.requires_grad_(), w.requires_grad_()
    value = llm_hgemm.linear_cross_entropy(poisoned, w, t, reduction=reduction)
    dx, dw = torch.autograd.grad(value, [poisoned, w], dl)
    value = value.detach()
    within(value[keep] if reduction == "none" else value, want[0])
    assert not dx[~keep].any()
    within(dx[keep], want[1])
    within(dw, want[2])
    (alone,) = torch.autograd.grad(llm_hgemm.linear_cross_entropy(poisoned.detach(), w, t, reduction=reduction), w, dl)
    within(alone, want[2])


class StatusWord:
    """The word that the torch functions give to their kernels, as an argument of the C calls."""

    def data_ptr(self):
        return _C.training_status_address()


def test_a_wait_that_ran_out_raises():
    inputs = ffn_inputs(390, 520, 712, 520, torch.bfloat16)
    training.check_status()
    want = llm_hgemm.gated_ffn(*inputs[:4])

    def stall():
        ffn_through_c(*inputs, 128, flags=capi.FLAG_TEST_INJECT_TX, status=StatusWord(), timeout_ns=50_000_000)
        torch.cuda.synchronize()

    stall()
    with pytest.raises(RuntimeError, match="earlier call of the training operators failed"):
        llm_hgemm.gated_ffn(*inputs[:4])
    assert torch.equal(llm_hgemm.gated_ffn(*inputs[:4]), want)     # raised once
    stall()
    with pytest.raises(RuntimeError, match="kernel of the training operators failed"):
        training.check_status()
    training.check_status()


def test_every_operator_raises_for_an_earlier_failure():
    x, gate, up, down, dy = ffn_inputs(40, 64, 136, 64, torch.float16)
    w, t = gate, torch.arange(40, device="cuda")
    x.requires_grad_()
    y, loss = llm_hgemm.gated_ffn(x, gate, up, down), llm_hgemm.linear_cross_entropy(x, w, t)
    word = ctypes.c_int32.from_address(_C.training_status_address())
    for call in (lambda: llm_hgemm.gated_ffn(x, gate, up, down), lambda: llm_hgemm.linear_cross_entropy(x, w, t),
                 lambda: llm_hgemm.orthogonalize(gate), lambda: torch.autograd.grad(y, x, dy, retain_graph=True),
                 lambda: torch.autograd.grad(loss, x, retain_graph=True)):
        word.value = capi.ERR_PIPELINE_TIMEOUT
        with pytest.raises(RuntimeError, match="earlier call"):
            call()
        assert word.value == 0
        call()


def test_values_negated_by_a_bit():
    """torch holds the imaginary part of a conjugate as its negative, by a bit of
    the tensor: as an input, and as the gradient that comes in behind one."""
    x, gate, up, down, dy = ffn_inputs(20, 64, 136, 72, torch.float16)
    neg = torch._neg_view
    assert neg(x).is_neg() and torch.equal(neg(x), -x)
    for k in range(4):
        args = [x, gate, up, down]
        args[k] = -args[k]
        want = llm_hgemm.gated_ffn(*args)
        args[k] = neg([x, gate, up, down][k])
        assert torch.equal(llm_hgemm.gated_ffn(*args), want)
    x.requires_grad_()
    y = llm_hgemm.gated_ffn(x, gate, up, down)
    (want,) = torch.autograd.grad(y, x, -dy, retain_graph=True)
    assert torch.equal(torch.autograd.grad(y, x, neg(dy))[0], want)
    assert torch.equal(llm_hgemm.orthogonalize(neg(gate)), llm_hgemm.orthogonalize(-gate))
    assert torch.equal(llm_hgemm.orthogonalize(neg(gate[:, :8])), llm_hgemm.orthogonalize(-gate[:, :8]))
    t = torch.arange(20, device="cuda")
    assert torch.equal(llm_hgemm.linear_cross_entropy(x, gate, neg(-t)), llm_hgemm.linear_cross_entropy(x, gate, t))
    loss = llm_hgemm.linear_cross_entropy(x, gate, t)
    (want,) = torch.autograd.grad(loss, x, torch.tensor(-3.0, device="cuda"), retain_graph=True)
    z = torch.complex(torch.zeros((), device="cuda"), loss).conj()
    assert torch.equal(torch.autograd.grad(3 * z.imag, x)[0], want)
