"""Training operators against their formulas in 64 bits (GPU), with the error
bounds of tests/training_reference.py: tile shapes, types, odd and ragged sizes,
ignored and invalid targets, strides, streams, captured graphs, differences."""

import os
import subprocess
import sys

import pytest
import torch
from torch import nn

import llm_hgemm
from llm_hgemm import capi, train_capi
from llm_hgemm.training import NEWTON_SCHULZ, TrainableSwiGLU
from tests import training_reference as ref
from tests.gpu_helpers import require_cuda

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
IDS = ["fp16", "bf16"]


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    require_cuda()


def normal(seed, *shape, dtype=torch.float16, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def ffn_inputs(tokens, hidden, inter, out, dtype, seed=1):
    return (normal(seed, tokens, hidden, dtype=dtype), normal(seed + 1, inter, hidden, dtype=dtype, scale=hidden ** -0.5),
            normal(seed + 2, inter, hidden, dtype=dtype, scale=hidden ** -0.5),
            normal(seed + 3, out, inter, dtype=dtype, scale=inter ** -0.5), normal(seed + 4, tokens, out, dtype=dtype))


def loss_inputs(tokens, hidden, vocab, dtype, ignore=-100, seed=1):
    w = normal(seed, vocab, hidden, dtype=dtype, scale=2 * hidden ** -0.5)
    gen = torch.Generator(device="cuda").manual_seed(seed + 7)
    t = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    x = (normal(seed + 1, tokens, hidden, dtype=dtype).float() + 2 * w[t].float()).to(dtype)
    t = torch.where(torch.rand(tokens, generator=gen, device="cuda") < 0.2, torch.full_like(t, ignore), t)
    return x, w, t


def within(got, want):
    value, err = want
    assert got.shape == value.shape
    off = (got.double() - value).abs()
    assert bool((off <= err).all()), f"off by {float((off / err).max()):.3g} times the bound"


def grads_of(y, leaves, dy):
    return torch.autograd.grad(y, leaves, dy)


# ------------------------------------------------------------ feed-forward ---

FFN_SIZES = [   # tokens, hidden, inter, out
    (1, 64, 128, 64),
    (1, 2560, 1024, 2560),
    (3, 8, 8, 8),
    (7, 72, 40, 136),
    (33, 264, 1000, 200),
    (127, 256, 688, 256),
    (129, 512, 320, 512),
    (257, 648, 1032, 640),
    (509, 1024, 2816, 1024),
    (1025, 768, 2048, 768),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("size", FFN_SIZES, ids=str)
def test_ffn(size, dtype):
    *leaves, dy = ffn_inputs(*size, dtype)
    want = ref.ffn(*leaves, dy)
    with torch.no_grad():
        within(llm_hgemm.gated_ffn(*leaves), want[0])
    leaves = [t.requires_grad_() for t in leaves]
    y = llm_hgemm.gated_ffn(*leaves)
    for got, w in zip([y.detach(), *grads_of(y, leaves, dy)], want):
        assert got.dtype == dtype
        within(got, w)


@pytest.mark.parametrize("size", [(5, 37, 53, 29), (130, 100, 300, 100)], ids=str)
def test_ffn_sizes_of_any_remainder(size):
    *leaves, dy = ffn_inputs(*size, torch.float16)
    leaves = [t.requires_grad_() for t in leaves]
    y = llm_hgemm.gated_ffn(*leaves)
    for got, w in zip([y.detach(), *grads_of(y, leaves, dy)], ref.ffn(*leaves, dy)):
        within(got, w)


TILES = [64, 128, 192, 256]


def stream():
    return torch.cuda.current_stream().cuda_stream


def with_workspace(name, args):
    """The call's workspace, filled with NaN; returned so that it lives on."""
    args.workspace_bytes = train_capi.workspace(name, args)
    ws = torch.full((args.workspace_bytes // 4,), float("nan"), device="cuda")
    args.workspace = ws.data_ptr() if args.workspace_bytes else None
    return ws


def ffn_through_c(x, gate, up, down, dy, tile, flags=0, splits=0, status=None, timeout_ns=0):
    """Both calls of the C ABI with a forced tile; outputs pre-filled with NaN."""
    (t, h), (i, _), o = x.shape, gate.shape, down.shape[0]
    like = lambda *s: torch.full(s, float("nan"), dtype=x.dtype, device="cuda")   # noqa: E731
    common = train_capi.Common(train_capi.BF16 if x.dtype == torch.bfloat16 else train_capi.F16, tile, flags, splits,
                               None if status is None else status.data_ptr(), timeout_ns)
    y, act, g, u, dg, du = like(t, o), like(t, i), like(t, i), like(t, i), like(t, i), like(t, i)
    dx, dgate, dup, ddown = like(t, h), like(i, h), like(i, h), like(o, i)
    p = lambda *ts: [a.data_ptr() for a in ts]   # noqa: E731
    f = train_capi.FfnForward(common, *p(x, gate, up, down, y, act, g, u), None, 0, t, h, i, o, h)
    ws = with_workspace("ffn_forward", f)
    assert train_capi.run("ffn_forward", f, stream()) == capi.OK
    b = train_capi.FfnBackward(common, *p(dy, x, gate, up, down, g, u, act, dg, du, dx, dgate, dup, ddown), None, 0,
                               t, h, i, o, h, o)
    ws2 = with_workspace("ffn_backward", b)
    assert train_capi.run("ffn_backward", b, stream()) == capi.OK
    if ws.numel() + ws2.numel():
        torch.cuda.synchronize()
        # Less than the call asks for is refused.
        for name, args in (("ffn_forward", f), ("ffn_backward", b)):
            if args.workspace_bytes:
                args.workspace_bytes -= 1
                assert train_capi.run(name, args, stream()) == capi.ERR_INVALID_ARGUMENT
    return y, dx, dgate, dup, ddown


@pytest.mark.parametrize("splits", [1, 2, 3, 5, 16])
@pytest.mark.parametrize("size", [(5, 72, 1000, 136), (130, 264, 584, 200), (300, 520, 1352, 640), (1100, 136, 584, 1352)],
                         ids=str)
def test_ffn_sums_in_parts(size, splits):
    """y and dx as sums of parts, whose borders fall inside either segment of dx's
    sum; of all tiles, or of those after the last full wave."""
    inputs = ffn_inputs(*size, torch.bfloat16)
    for tile in (64, 192, 128 | train_capi.TILE_PAIR):
        for got, w in zip(ffn_through_c(*inputs, tile, splits=splits), ref.ffn(*inputs)):
            within(got, w)


@pytest.mark.parametrize("pair", [0, train_capi.TILE_PAIR], ids=["single", "pair"])
@pytest.mark.parametrize("width", TILES)
def test_ffn_every_tile(width, pair):
    """Each tile shape of the GEMM, on sizes whose edges fall inside tiles and
    with more tiles than one wave for the narrow ones."""
    inputs = ffn_inputs(390, 1352, 1992, 1096, torch.bfloat16)
    for got, w in zip(ffn_through_c(*inputs, width | pair), ref.ffn(*inputs)):
        within(got, w)


def test_ffn_only_the_wanted_gradients():
    x, gate, up, down, dy = ffn_inputs(70, 128, 256, 128, torch.bfloat16)
    want = ref.ffn(x, gate, up, down, dy)
    for wanted in ([0], [1], [3], [0, 2], [1, 2, 3]):
        tensors = [t.detach().clone().requires_grad_(k in wanted) for k, t in enumerate((x, gate, up, down))]
        y = llm_hgemm.gated_ffn(*tensors)
        y.backward(dy)
        for k, t in enumerate(tensors):
            if k in wanted:
                within(t.grad, want[1 + k])
            else:
                assert t.grad is None


def test_ffn_strides_and_leading_dimensions():
    x, gate, up, down, dy = ffn_inputs(60, 128, 256, 64, torch.float16)
    want = ref.ffn(x, gate, up, down, dy)
    wide = normal(9, 60, 300)
    wide[:, 40:168] = x                       # rows 300 apart, 16-byte aligned
    odd = normal(9, 60, 301)
    odd[:, 41:169] = x                        # rows 301 apart, at an odd offset
    turned = x.t().contiguous().t()           # columns unit apart in the other dimension
    gate_turned = gate.t().contiguous().t()
    for v in (wide[:, 40:168], odd[:, 41:169], turned):
        within(llm_hgemm.gated_ffn(v, gate_turned, up, down), want[0])
    cube = x.view(3, 4, 5, 128).requires_grad_()
    y = llm_hgemm.gated_ffn(cube, gate, up, down)
    assert y.shape == (3, 4, 5, 64)
    (dx,) = torch.autograd.grad(y, cube, dy.view(3, 4, 5, 64))
    within(dx.view(60, 128), want[1])
    # A broadcast incoming gradient (stride 0).
    (dx,) = torch.autograd.grad(llm_hgemm.gated_ffn(cube, gate, up, down).sum(), cube)
    within(dx.view(60, 128), ref.ffn(x, gate, up, down, torch.ones_like(dy))[1])


def test_ffn_no_tokens_and_shared_weights():
    x, gate, _, down, dy = ffn_inputs(20, 64, 128, 64, torch.float16)
    none = x[:0].clone().requires_grad_()
    g = gate.clone().requires_grad_()
    y = llm_hgemm.gated_ffn(none, g, g, down)
    assert y.shape == (0, 64)
    y.sum().backward()
    assert none.grad.shape == (0, 64) and not g.grad.any()
    # gate and up the same tensor: both gradients add up.
    g = gate.clone().requires_grad_()
    llm_hgemm.gated_ffn(x, g, g, down).backward(dy)
    want = ref.ffn(x, gate, gate, down, dy)
    (a, ea), (b, eb) = want[2], want[3]
    within(g.grad, (a + b, ea + eb + ref.unit(torch.float16) * (a + b).abs()))


def test_ffn_special_values_stay_in_their_rows():
    x, gate, up, down, _ = ffn_inputs(130, 64, 128, 64, torch.float16)
    clean = llm_hgemm.gated_ffn(x, gate, up, down)
    x[5] = float("nan")
    x[128, 3] = float("inf")
    y = llm_hgemm.gated_ffn(x, gate, up, down)
    assert y[5].isnan().all() and not y[128].isfinite().all()
    rest = [r for r in range(130) if r not in (5, 128)]
    assert torch.equal(y[rest], clean[rest])
    # Large negative pre-activations: silu is 0, not NaN.
    big = torch.full((4, 64), 100.0, dtype=torch.float16, device="cuda")
    y = llm_hgemm.gated_ffn(big, -torch.ones_like(gate), torch.ones_like(up), down)
    assert bool((y == 0).all())


def test_ffn_against_differences():
    """The directional derivative by central differences of the 64-bit formula
    at the same points: the two agree to the bound and the difference's own error."""
    x, gate, up, down, dy = ffn_inputs(9, 40, 48, 32, torch.float16)
    leaves = [t.requires_grad_() for t in (x, gate, up, down)]
    grads = grads_of(llm_hgemm.gated_ffn(*leaves), leaves, dy)
    want = ref.ffn(*leaves, dy)
    for k in range(4):
        direction = normal(50 + k, *leaves[k].shape).double()
        step = 1e-4

        def f(sign):
            moved = [t.detach().double() + (sign * step * direction if j == k else 0) for j, t in enumerate(leaves)]
            pre = moved[0] @ moved[1].T
            return ((torch.nn.functional.silu(pre) * (moved[0] @ moved[2].T)) @ moved[3].T * dy.double()).sum()

        diff = (f(1) - f(-1)) / (2 * step)
        # Third derivatives are of order one here: the difference is off by about step^2 |d|^3.
        slack = (want[1 + k][1] * direction.abs()).sum() + 1e-3 * (1 + diff.abs())
        assert abs((grads[k].double() * direction).sum() - diff) <= slack


# ------------------------------------------------------------ cross entropy ---

LOSS_SIZES = [   # tokens, hidden, vocab
    (1, 8, 2),
    (1, 64, 1),
    (2, 72, 31),
    (17, 136, 257),
    (24, 256, 4001),
    (129, 64, 1000),
    (300, 264, 513),
    (1, 2560, 12345),
    (257, 520, 10007),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("size", LOSS_SIZES, ids=str)
def test_loss(size, reduction, dtype):
    x, w, t = loss_inputs(*size, dtype)
    t[0] = size[2] - 1          # one target at least, in the last column
    dl = (torch.rand(size[0], device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 100
          if reduction == "none" else torch.tensor(64.0, device="cuda"))
    want = ref.loss(x, w, t, reduction, -100, dl)
    within(llm_hgemm.linear_cross_entropy(x, w, t, reduction=reduction), want[0])
    x.requires_grad_(), w.requires_grad_()
    value = llm_hgemm.linear_cross_entropy(x, w, t, reduction=reduction)
    assert value.dtype == torch.float32
    for got, v in zip([value.detach(), *grads_of(value, [x, w], dl)], want):
        within(got, v)


def loss_through_c(x, w, t, dl, tile=0, piece=0, reduction=train_capi.LOSS_MEAN, splits=0):
    """Forward and backward through the C ABI, outputs and workspaces pre-filled with NaN."""
    n, h = x.shape
    v = w.shape[0]
    common = train_capi.Common(train_capi.BF16 if x.dtype == torch.bfloat16 else train_capi.F16, tile, 0, splits)
    loss = torch.full((n if reduction == train_capi.LOSS_NONE else 1,), float("nan"), device="cuda")
    lse = torch.full((n,), float("nan"), device="cuda")
    f = train_capi.LossForward(common, x.data_ptr(), w.data_ptr(), t.data_ptr(), loss.data_ptr(), lse.data_ptr(), None, 0,
                               n, h, v, h, -100, reduction, 0)
    keep = [with_workspace("loss_forward", f)]
    assert train_capi.run("loss_forward", f, stream()) == capi.OK
    dx, dw = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))
    b = train_capi.LossBackward(common, x.data_ptr(), w.data_ptr(), t.data_ptr(), lse.data_ptr(), dl.data_ptr(),
                                dx.data_ptr(), dw.data_ptr(), None, 0, n, h, v, h, -100, piece, reduction, 0)
    keep.append(with_workspace("loss_backward", b))
    assert train_capi.run("loss_backward", b, stream()) == capi.OK
    torch.cuda.synchronize()
    return loss, dx, dw


@pytest.mark.parametrize("splits", [1, 2, 7, 16])
@pytest.mark.parametrize("piece", [64, 320, 1000, 5000])
def test_loss_sums_in_parts(piece, splits):
    """dx in pieces of the vocabulary and parts of each, the last piece short."""
    x, w, t = loss_inputs(70, 136, 2100, torch.bfloat16)
    dl = torch.tensor([1.0], device="cuda")
    want = ref.loss(x, w, t, "sum", -100, dl)
    got = loss_through_c(x, w, t, dl, piece=piece, reduction=train_capi.LOSS_SUM, splits=splits)
    for g, v in zip((got[0][0], got[1], got[2]), want):
        within(g, v)


def test_loss_workspace_holds_one_piece():
    a = train_capi.LossBackward(tokens=1000, hidden=64, vocab=150000, dx=1 << 20)
    # At most 96 MB of 16-bit logit gradients (and the sums of dx), not the 300 MB of all.
    assert 0 < train_capi.workspace("loss_backward", a) < 140 << 20
    a.tokens = 0
    assert train_capi.workspace("loss_backward", a) == 0


@pytest.mark.parametrize("pair", [0, train_capi.TILE_PAIR], ids=["single", "pair"])
@pytest.mark.parametrize("width", TILES)
def test_loss_every_tile(width, pair):
    x, w, t = loss_inputs(390, 328, 20011, torch.float16)
    dl = torch.tensor([32.0], device="cuda")
    want = ref.loss(x, w, t, "mean", -100, dl)
    got = loss_through_c(x, w, t, dl, width | pair)
    for g, v in zip((got[0][0], got[1], got[2]), want):
        within(g, v)


@pytest.mark.parametrize("piece", [8, 264, 1000, 2049, 5000, 100000])
def test_loss_pieces_of_the_vocabulary(piece):
    x, w, t = loss_inputs(200, 136, 4999, torch.bfloat16)
    dl = torch.tensor([1.0], device="cuda")
    want = ref.loss(x, w, t, "sum", -100, dl)
    got = loss_through_c(x, w, t, dl, piece=piece, reduction=train_capi.LOSS_SUM)
    for g, v in zip((got[0][0], got[1], got[2]), want):
        within(g, v)


def test_loss_odd_hidden_size_strides_and_int32_targets():
    x, w, t = loss_inputs(45, 37, 300, torch.float16)
    dl = torch.tensor(8.0, device="cuda")
    want = ref.loss(x, w, t, "sum", -100, dl)
    wide = normal(3, 45, 99)
    wide[:, 11:48] = x
    a, b = wide[:, 11:48].detach().view(3, 15, 37).requires_grad_(), w.requires_grad_()
    value = llm_hgemm.linear_cross_entropy(a, b, t.int().view(3, 15), reduction="sum")
    dx, dw = grads_of(value, [a, b], dl)
    assert dx.shape == (3, 15, 37)
    for got, v in zip((value.detach(), dx.reshape(45, 37), dw), want):
        within(got, v)
    each = llm_hgemm.linear_cross_entropy(a.detach(), b.detach(), t.view(3, 15), reduction="none")
    assert each.shape == (3, 15)


def test_loss_ignored_and_invalid_targets():
    x, w, t = loss_inputs(40, 64, 500, torch.float16)
    x.requires_grad_(), w.requires_grad_()
    nothing = torch.full_like(t, -100)
    for reduction, want in (("mean", float("nan")), ("sum", 0.0)):
        value = llm_hgemm.linear_cross_entropy(x, w, nothing, reduction=reduction)
        assert torch.equal(value, torch.tensor(want, device="cuda")) or value.isnan() and want != want
        dx, dw = grads_of(value, [x, w], torch.ones((), device="cuda"))
        assert not dx.any() and not dw.any()
    # An ignored row may hold anything.
    poisoned = x.detach().clone()
    poisoned[3] = float("nan")
    t[3] = -100
    keep = torch.arange(40, device="cuda") != 3
    p = poisoned.requires_grad_()
    value = llm_hgemm.linear_cross_entropy(p, w, t, reduction="sum")
    want = ref.loss(x.detach()[keep], w, t[keep], "sum", -100, torch.ones((), device="cuda"))
    within(value.detach(), want[0])
    (dx,) = torch.autograd.grad(value, p)
    assert not dx[3].any()
    within(dx[keep], want[1])
    # Another ignore_index, among the valid classes.
    got = llm_hgemm.linear_cross_entropy(x.detach(), w.detach(), t.clamp(min=0), reduction="none", ignore_index=0)
    assert bool((got[t.clamp(min=0) == 0] == 0).all())
    # Outside the vocabulary: NaN for that token, the others as they were.
    for bad in (500, -1, 2 ** 40):
        t2 = t.clone()
        t2[7] = bad
        each = llm_hgemm.linear_cross_entropy(x.detach(), w.detach(), t2, reduction="none")
        assert each[7].isnan() and int(each.isnan().sum()) == 1
        dx, = torch.autograd.grad(llm_hgemm.linear_cross_entropy(x, w.detach(), t2, reduction="sum"), x)
        assert dx[7].isnan().all() and int(dx.isnan().any(dim=1).sum()) == 1


def test_loss_extreme_logits_and_gradients():
    """Logits of +-3000, rows with one certain class, and incoming gradients over
    16 orders of magnitude or zero."""
    w = torch.zeros(300, 64, dtype=torch.float16, device="cuda")
    w[:, 0] = torch.linspace(-50, 50, 300, device="cuda").half()
    x = torch.zeros(6, 64, dtype=torch.float16, device="cuda")
    x[:, 0] = torch.tensor([60.0, -60.0, 0.0, 1e-3, 20.0, -1.0], device="cuda").half()
    t = torch.tensor([299, 0, 5, 7, 299, 1], device="cuda")
    x.requires_grad_(), w.requires_grad_()
    for dl in (torch.tensor([1e4, 1e-12, 1.0, 3.0, 1e-3, 0.5], device="cuda"), torch.zeros(6, device="cuda")):
        value = llm_hgemm.linear_cross_entropy(x, w, t, reduction="none")
        want = ref.loss(x, w, t, "none", -100, dl)
        for got, v in zip([value.detach(), *grads_of(value, [x, w], dl)], want):
            within(got, v)


def test_one_token_without_a_token_dimension():
    x, gate, up, down, dy = ffn_inputs(1, 64, 128, 72, torch.float16)
    v = x[0].clone().requires_grad_()
    y = llm_hgemm.gated_ffn(v, gate, up, down)
    want = ref.ffn(x, gate, up, down, dy)
    assert y.shape == (72,)
    (dx,) = torch.autograd.grad(y, v, dy[0])
    within(y.detach()[None], want[0])
    within(dx[None], want[1])
    w = normal(3, 90, 64)
    t = torch.tensor(5, device="cuda")
    each = llm_hgemm.linear_cross_entropy(v, w, t, reduction="none")
    assert each.shape == ()
    (dx,) = torch.autograd.grad(each, v, torch.tensor(2.0, device="cuda"))
    want = ref.loss(x, w, t[None], "none", -100, torch.tensor([2.0], device="cuda"))
    within(each.detach()[None], want[0])
    within(dx[None], want[1])


def test_loss_no_tokens():
    w = normal(1, 50, 64).requires_grad_()
    x = normal(2, 0, 64).requires_grad_()
    t = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert llm_hgemm.linear_cross_entropy(x, w, t).isnan()
    value = llm_hgemm.linear_cross_entropy(x, w, t, reduction="sum")
    value.backward()
    assert value == 0 and not w.grad.any() and x.grad.shape == (0, 64)
    assert llm_hgemm.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)


def test_loss_against_differences():
    x, w, t = loss_inputs(11, 40, 77, torch.float16)
    x.requires_grad_(), w.requires_grad_()
    dl = torch.ones((), device="cuda")
    grads = grads_of(llm_hgemm.linear_cross_entropy(x, w, t), [x, w], dl)
    want = ref.loss(x, w, t, "mean", -100, dl)
    for k in range(2):
        d = normal(60 + k, *(x, w)[k].shape).double()

        def f(sign):
            a, b = (v.detach().double() + (sign * 1e-4 * d if j == k else 0) for j, v in enumerate((x, w)))
            return torch.nn.functional.cross_entropy(a @ b.T, t)

        diff = (f(1) - f(-1)) / 2e-4
        slack = (want[1 + k][1] * d.abs()).sum() + 1e-3 * (1 + diff.abs())
        assert abs((grads[k].double() * d).sum() - diff) <= slack


# ------------------------------------------------------ orthogonalised update ---

ORTH_SIZES = [(1, 1), (1, 9), (9, 1), (8, 8), (16, 40), (96, 256), (256, 96), (129, 131), (333, 1001), (513, 64),
              (1000, 250), (512, 512)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("size", ORTH_SIZES, ids=str)
def test_orthogonalize(size, dtype):
    g = normal(5, *size, dtype=dtype, scale=1e-3)
    value, err = ref.orthogonalize(g, 5, NEWTON_SCHULZ, 1e-7)
    got = llm_hgemm.orthogonalize(g)
    assert got.shape == g.shape and got.dtype == dtype and got.is_contiguous()
    assert float(torch.linalg.vector_norm(got.double() - value)) <= err


@pytest.mark.parametrize("turn", [False, True], ids=["wide", "tall"])
@pytest.mark.parametrize("size", [(1, 640), (2, 641), (17, 1280), (128, 1283), (31, 2560), (96, 2600), (65, 5119),
                                  (128, 9728), (48, 10240), (33, 10241), (128, 64), (129, 300)], ids=str)
def test_orthogonalize_one_launch_and_its_limits(size, turn):
    """A shorter side of at most 128 is one launch of 1 to 16 CTAs a matrix; around its limits."""
    g = normal(11, 3, *(size[::-1] if turn else size), dtype=torch.bfloat16)
    out = llm_hgemm.orthogonalize(g)
    for k in range(3):
        value, err = ref.orthogonalize(g[k], 5, NEWTON_SCHULZ, 1e-7)
        assert float(torch.linalg.vector_norm(out[k].double() - value)) <= err


@pytest.mark.parametrize("splits", [0, 1, 2, 5])
@pytest.mark.parametrize("tile", [0, 64, 128, 256 | train_capi.TILE_PAIR])
@pytest.mark.parametrize("size", [(140, 1100), (1500, 1010), (1003, 2100)], ids=str)
def test_orthogonalize_triangles_and_parts(size, tile, splits):
    """Symmetric products by their upper triangle, the others' last wave in parts."""
    g = normal(13, *size)
    value, err = ref.orthogonalize(g, 5, NEWTON_SCHULZ, 1e-7)
    out = torch.full_like(g, float("nan"))
    a = train_capi.Orthogonalize(train_capi.Common(train_capi.F16, tile, 0, splits), g.data_ptr(), out.data_ptr(), None,
                                 0, 1, *size, size[1], 0, 5, 0, *NEWTON_SCHULZ, 0.0, 1e-7)
    ws = with_workspace("orthogonalize", a)
    # X twice and two square matrices, rows padded to 64 elements.
    assert ws.numel() * 2 >= 2 * size[0] * size[1] + 2 * min(size) ** 2
    assert train_capi.run("orthogonalize", a, stream()) == capi.OK
    assert float(torch.linalg.vector_norm(out.double() - value)) <= err
    a.workspace_bytes -= 1
    assert train_capi.run("orthogonalize", a, stream()) == capi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("ctas", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("size", [(40, 300), (300, 40), (128, 1), (128, 600), (600, 128)], ids=str)
def test_orthogonalize_every_cluster(size, ctas):
    """Every size of cluster, also with CTAs that hold no column at all."""
    g = normal(12, *size)
    value, err = ref.orthogonalize(g, 5, NEWTON_SCHULZ, 1e-7)
    out = torch.full_like(g, float("nan"))
    a = train_capi.Orthogonalize(train_capi.Common(train_capi.F16, 0, 0, ctas), g.data_ptr(), out.data_ptr(), None, 0,
                                 1, *size, size[1], 0, 5, 0, *NEWTON_SCHULZ, 0.0, 1e-7)
    assert train_capi.workspace("orthogonalize", a) == 0
    assert train_capi.run("orthogonalize", a, stream()) == capi.OK
    assert float(torch.linalg.vector_norm(out.double() - value)) <= err


@pytest.mark.parametrize("batch", [(1,), (3,), (4,), (5,), (2, 3)], ids=str)
def test_orthogonalize_batches_and_strides(batch):
    for size in ((40, 77), (150, 177)):
        g = normal(6, *batch, *size, scale=0.1)
        got = llm_hgemm.orthogonalize(g)
        for k, m in enumerate(g.view(-1, *size)):
            assert torch.equal(got.view(-1, *size)[k], llm_hgemm.orthogonalize(m))
    wide = normal(7, *batch, 50, 200, scale=0.1)
    assert torch.equal(llm_hgemm.orthogonalize(wide[..., 3:43, 5:82]), llm_hgemm.orthogonalize(wide[..., 3:43, 5:82].contiguous()))
    assert torch.equal(llm_hgemm.orthogonalize(g.mT), llm_hgemm.orthogonalize(g.mT.contiguous()))


def test_orthogonalize_steps_coefficients_and_zeros():
    g = normal(8, 60, 90, dtype=torch.bfloat16)
    for steps, co in ((0, NEWTON_SCHULZ), (1, NEWTON_SCHULZ), (10, (1.5, -0.5, 0.0))):
        value, err = ref.orthogonalize(g, steps, co, 1e-7)
        got = llm_hgemm.orthogonalize(g, steps=steps, coefficients=co)
        assert float(torch.linalg.vector_norm(got.double() - value)) <= err
    zero = torch.zeros(30, 50, dtype=torch.float16, device="cuda")
    assert not llm_hgemm.orthogonalize(zero).any()
    # Far outside FP32's squares, and with eps as the whole norm.
    for scale in (1e30, 1e-30):
        h = (normal(9, 24, 32, dtype=torch.bfloat16).float() * scale).bfloat16()
        value, err = ref.orthogonalize(h, 5, NEWTON_SCHULZ, 0.0)
        assert float(torch.linalg.vector_norm(llm_hgemm.orthogonalize(h, eps=0.0).double() - value)) <= err
    assert llm_hgemm.orthogonalize(g.requires_grad_()).requires_grad is False
    assert llm_hgemm.orthogonalize(zero[:0]).shape == (0, 50)


@pytest.mark.parametrize("size", [(8, 24), (9, 23), (136, 200)], ids=str)
def test_orthogonalize_of_the_smallest_and_largest_elements(size):
    """Without eps the result does not depend on a power of two in g, over all of
    BF16's normal numbers: at the first scale 256 / norm is beyond FP32 (elements
    of 2^-126 to 2^-123, a few of them in the large matrix)."""
    g = normal(11, *size, dtype=torch.bfloat16)
    g = torch.where(g < 0, -1.0, 1.0).bfloat16() * g.abs().clamp(0.5, 4)
    if g.numel() > 1000:
        keep = torch.rand(size, generator=torch.Generator(device="cuda").manual_seed(12), device="cuda") < 0.005
        g = torch.where(keep, g, torch.zeros_like(g))
    assert float(g.double().norm()) * 2.0 ** -125 < 2.0 ** -120
    want = llm_hgemm.orthogonalize(g, eps=0.0)
    assert bool(want.isfinite().all())
    for exponent in (-125, -100, 100, 125):
        h = (g.double() * 2.0 ** exponent).bfloat16()
        assert torch.equal(llm_hgemm.orthogonalize(h, eps=0.0), want)


@pytest.mark.parametrize("pair", [0, train_capi.TILE_PAIR], ids=["single", "pair"])
@pytest.mark.parametrize("width", TILES)
@pytest.mark.parametrize("size", [(300, 700), (700, 300)], ids=str)
def test_orthogonalize_every_tile(size, width, pair):
    g = normal(10, *size)
    value, err = ref.orthogonalize(g, 5, NEWTON_SCHULZ, 1e-7)
    out = torch.full_like(g, float("nan"))
    a = train_capi.Orthogonalize(train_capi.Common(train_capi.F16, width | pair), g.data_ptr(), out.data_ptr(), None, 0,
                                 1, *size, size[1], 0, 5, 0, *NEWTON_SCHULZ, 0.0, 1e-7)
    ws = with_workspace("orthogonalize", a)
    assert ws.numel() > 0
    assert train_capi.run("orthogonalize", a, stream()) == capi.OK
    assert float(torch.linalg.vector_norm(out.double() - value)) <= err


def test_orthogonalize_many_clusters_on_two_streams():
    """More clusters than fit the GPU at once, of two calls at the same time."""
    g = [normal(14 + k, 40, *size) for k, size in enumerate(((16, 2100), (100, 700)))]
    want = [llm_hgemm.orthogonalize(t) for t in g]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in g]
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(llm_hgemm.orthogonalize(g[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert torch.equal(want[k][7], llm_hgemm.orthogonalize(g[k][7]))
        for t in got[k]:
            assert torch.equal(t, want[k])


# -------------------------------------------------------- how they are called ---

def run_all(x, gate, up, down, w, t, dy):
    y = llm_hgemm.gated_ffn(x, gate, up, down)
    value = llm_hgemm.linear_cross_entropy(y, w, t)
    grads = torch.autograd.grad(value, [x, gate, up, down, w])
    return [y.detach(), value.detach(), *grads, llm_hgemm.orthogonalize(grads[1])]


def all_inputs(tokens=90, seed=1):
    x, gate, up, down, dy = ffn_inputs(tokens, 128, 320, 128, torch.bfloat16, seed)
    _, w, t = loss_inputs(tokens, 128, 3001, torch.bfloat16, seed=seed + 20)
    return [v.requires_grad_() for v in (x, gate, up, down, w)][:4] + [w, t, dy]


def test_same_result_every_time_and_on_another_stream():
    inputs = all_inputs()
    first = run_all(*inputs)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        again = run_all(*inputs)
    other.synchronize()
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    sets = [all_inputs(seed=s) for s in (1, 100)]
    want = [run_all(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = run_all(*sets[k])
    torch.cuda.synchronize()
    for k in range(2):
        for a, b in zip(want[k], got[k]):
            assert torch.equal(a, b)


def test_captured_and_replayed():
    """A whole step in a CUDA graph, replayed on new inputs in place, twice."""
    inputs = all_inputs()
    fresh = [all_inputs(seed=s) for s in (40, 80)]
    want = [run_all(*f) for f in fresh]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_all(*inputs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run_all(*inputs)
    for f, w in zip(fresh, want):
        with torch.no_grad():
            for dst, src in zip(inputs, f):
                dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, w):
            assert torch.equal(a, b)


@pytest.mark.parametrize("what", ["ffn", "loss"])
def test_captured_backward_beside_an_eager_graph_is_refused(what):
    x, gate, up, down, w, t, dy = all_inputs()

    def call():
        if what == "loss":
            return llm_hgemm.linear_cross_entropy(x, w, t), [x, w]
        return llm_hgemm.gated_ffn(x, gate, up, down).float().sum(), [x, gate, up, down]

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, leaves = call()
            out = torch.autograd.grad(y, leaves)
        return graph, out

    want = torch.autograd.grad(*call())
    eager, _ = call()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        capture()
    torch.cuda.synchronize()
    for got, v in zip(torch.autograd.grad(eager, call()[1]), want):   # the eager graph still works
        assert torch.equal(got, v)
    del eager
    graph, out = capture()
    graph.replay()
    torch.cuda.synchronize()
    for got, v in zip(out, want):
        assert torch.equal(got, v)


FIRST_CALL = """
import torch, llm_hgemm
gen = torch.Generator(device="cuda").manual_seed(1)
r = lambda *s: torch.randn(s, generator=gen, device="cuda").half() / 8
x, gate, up, down, w, g = r(40, 64), r(96, 64), r(96, 64), r(64, 96), r(500, 64), r(200, 300)
t = torch.arange(40, device="cuda")
run = lambda: (llm_hgemm.gated_ffn(x, gate, up, down), llm_hgemm.linear_cross_entropy(x, w, t),
               llm_hgemm.orthogonalize(g), llm_hgemm.orthogonalize(g[:50]))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, run()))
print("same")
"""


def test_first_call_of_a_process_captured():
    done = subprocess.run([sys.executable, "-c", FIRST_CALL], capture_output=True, text=True, timeout=300,
                          env={**os.environ, "PYTHONPATH": os.pathsep.join(p for p in sys.path if p)})
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


def test_ffn_past_32_bits():
    """tokens x inter beyond 2^31: the last rows, and the last columns' weight
    gradients (of the last rows alone, so that the bound of 131080 FP32 additions
    stays below the values)."""
    tokens, hidden, inter = 131080, 64, 17408
    x, gate, up, down, dy = ffn_inputs(tokens, hidden, inter, 64, torch.float16)
    dy[:-64] = 0
    leaves = [v.requires_grad_() for v in (x, gate, up, down)]
    y = llm_hgemm.gated_ffn(*leaves)
    dx, dgate, dup, ddown = torch.autograd.grad(y, leaves, dy)
    want = ref.ffn(x[-40:], gate, up, down, dy[-40:])
    within(y.detach()[-40:], want[0])
    within(dx[-40:], want[1])
    assert not dx[:-64].any()
    last = ref.ffn(x, gate[-8:], up[-8:], down[:, -8:], dy)
    within(dgate[-8:], last[2])
    within(dup[-8:], last[3])
    within(ddown[:, -8:], last[4])


def test_loss_past_32_bits():
    """vocabulary x hidden beyond 2^31. All of W but its first and last 1000 rows is
    zero: there the logits are 0, and one entry with probability stands for them."""
    tokens, hidden, vocab, ends = 16, 1024, 2100000, 1000
    x = normal(1, tokens, hidden, dtype=torch.bfloat16, scale=0.1)
    some = normal(2, 2 * ends, hidden, dtype=torch.bfloat16)
    w = torch.zeros(vocab, hidden, dtype=torch.bfloat16, device="cuda")
    w[:ends], w[-ends:] = some[:ends], some[ends:]
    t = torch.where(torch.arange(tokens, device="cuda") % 2 == 0, 7, vocab - 7)
    x.requires_grad_(), w.requires_grad_()
    value = llm_hgemm.linear_cross_entropy(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(value, [x, w])
    z = x.detach().double() @ some.double().T
    lse = torch.log(z.exp().sum(1) + (vocab - 2 * ends))
    at = torch.where(t < ends, t, t - vocab + 2 * ends)
    d = torch.exp(z - lse[:, None])
    d[torch.arange(tokens, device="cuda"), at] -= 1
    # Relative error of a probability: FP32 sums of 1024 products, at most
    # (1024 + 8) 2^-23 sum |x w|, for the logit and the statistics; 2^-24 for each of
    # at most 40 + V / 32 additions; some 2^-20 for exp. Then dz is rounded once.
    logit = 1032 * 2.0 ** -23 * float((x.detach().double().abs() @ some.double().abs().T).max())
    off = 2 * logit + (40 + vocab / 32) * 2.0 ** -24 + 2.0 ** -20
    assert off < 0.06
    total = (lse - z.gather(1, at[:, None])[:, 0]).sum()
    assert abs(float(value.detach().double() - total)) <= tokens * (off + 2.0 ** -20 * float(lse.max()))
    for got, p, q in ((dx, d, some.double()), (torch.cat([dw[:ends], dw[-ends:]]), d.T, x.detach().double())):
        v, most = p @ q, p.abs() @ q.abs()
        err = (off + 2.0 ** -8 + 1032 * 2.0 ** -23) * most + 2.0 ** -8 * v.abs() * 1.1 + 1e-30
        assert bool(((got.double() - v).abs() <= err).all())
    # A row of the zeros: -p of that column times x, in every one of them.
    p0 = torch.exp(-lse)
    v, most = p0 @ x.detach().double(), p0 @ x.detach().double().abs()
    err = (off + 2.0 ** -7) * most + 2.0 ** -8 * v.abs()
    for row in (ends, vocab // 2, vocab - ends - 1):
        assert bool(((dw[row].double() - v).abs() <= err).all())


def test_orthogonalize_past_32_bits():
    """rows x cols beyond 2^31, zero but for the first and last 1000 rows: their
    update is that of the 2000 rows alone."""
    rows, cols, ends = 16000000, 136, 1000
    some = normal(3, 2 * ends, cols, dtype=torch.bfloat16)
    g = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    g[:ends], g[-ends:] = some[:ends], some[ends:]
    value, err = ref.orthogonalize(some, 5, NEWTON_SCHULZ, 1e-7)
    got = llm_hgemm.orthogonalize(g)
    assert not got[ends:-ends].any()
    got = torch.cat([got[:ends], got[-ends:]])
    assert float(torch.linalg.vector_norm(got.double() - value)) <= err


def test_injected_stall_times_out_and_context_survives():
    inputs = ffn_inputs(390, 520, 712, 520, torch.bfloat16)
    for tile in (128, 128 | train_capi.TILE_PAIR):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        ffn_through_c(*inputs, tile, flags=capi.FLAG_TEST_INJECT_TX, status=status, timeout_ns=50_000_000)
        torch.cuda.synchronize()
        assert int(status) == capi.ERR_PIPELINE_TIMEOUT
        for got, w in zip(ffn_through_c(*inputs, tile), ref.ffn(*inputs)):
            within(got, w)
    assert train_capi.read_status() == (capi.OK, 0)


def test_second_derivatives_and_changed_weights_are_refused():
    x, gate, up, down, w, t, dy = all_inputs()
    y = llm_hgemm.gated_ffn(x, gate, up, down)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(llm_hgemm.linear_cross_entropy(x, w, t), x, create_graph=True)
    y = llm_hgemm.gated_ffn(x, gate, up, down)
    with torch.no_grad():
        gate.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dy)


def test_a_training_step_of_a_small_model():
    """Module, head loss and orthogonalised update together, against the same
    step on the stock modules: the gradients to the formula's bounds."""
    torch.manual_seed(0)
    parts = [nn.Linear(128, 320, bias=False), nn.Linear(128, 320, bias=False), nn.Linear(320, 128, bias=False)]
    block = TrainableSwiGLU(*parts).to("cuda", torch.bfloat16)
    assert sorted(block.state_dict()) == ["down_proj.weight", "gate_proj.weight", "up_proj.weight"]
    head = normal(3, 1001, 128, dtype=torch.bfloat16, scale=0.1).requires_grad_()
    x = normal(4, 2, 35, 128, dtype=torch.bfloat16)
    t = torch.randint(0, 1001, (2, 35), device="cuda")
    for _ in range(2):
        y = block(x)
        y.retain_grad()
        value = llm_hgemm.linear_cross_entropy(y, head, t)
        value.backward()
        weights = [block.gate_proj.weight, block.up_proj.weight, block.down_proj.weight]
        want = ref.loss(y.detach().view(70, 128), head, t.view(70), "mean", -100, torch.ones((), device="cuda"))
        for got, v in zip((value.detach(), y.grad.view(70, 128), head.grad), want):
            within(got, v)
        for p, v in zip(weights, ref.ffn(x.view(70, 128), *weights, y.grad.view(70, 128))[2:]):
            within(p.grad, v)
        with torch.no_grad():
            for p in weights + [head]:
                update = llm_hgemm.orthogonalize(p.grad)
                value_, err = ref.orthogonalize(p.grad, 5, NEWTON_SCHULZ, 1e-7)
                assert float(torch.linalg.vector_norm(update.double() - value_)) <= err
                p -= 0.02 * update
                p.grad = None


def test_model_training_step():
    """A small decoder with ``trainable_mlps`` and ``linear_cross_entropy``: each
    FP16 model's gradients against the FP32 model's. Ours round the MLP three
    times (the product and its two derivatives) where the stock model rounds
    four times, and the logits never: no parameter may be further off than 1.5
    times the stock model's worst."""
    import importlib.util

    from tests.conftest import PKG

    spec = importlib.util.spec_from_file_location("model_check", PKG / "model_check.py")
    mc = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mc)
    args = mc.parser().parse_args(["--train", "--layers", "2", "--hidden", "256", "--intermediate", "704", "--heads", "4",
                                   "--kv-heads", "2", "--head-dim", "64", "--vocab", "1000", "--prefill-tokens", "96",
                                   "--context", "64"])
    res = mc.train_check(args)
    assert res["mlps"] == 2 and res["updates"]["matrices"] == 6
    assert res["hgemm"]["worst_gradient_relative_l2"] <= 1.5 * res["stock"]["worst_gradient_relative_l2"], res
    # Losses of about 7, each in FP32 from FP16 activations: 2^-11 relative is a wide margin.
    assert abs(res["hgemm"]["loss"] - res["fp32_loss"]) <= 2 ** -11 * res["fp32_loss"], res
