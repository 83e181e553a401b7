"""Training operators on the host (CPU): what the Python layer and the C ABI
refuse, the struct mirrors, and the 64-bit formulas the GPU tests compare with
(against torch's own autograd and a singular value decomposition)."""

import ctypes

import pytest
import torch
from torch import nn

import llm_hgemm
from llm_hgemm import capi, train_capi
from llm_hgemm.training import NEWTON_SCHULZ, TrainableSwiGLU
from tests import training_reference as ref


def test_struct_layouts():
    """Sizes of include/hgemm_sm100_train.h's structs on x86-64."""
    assert ctypes.sizeof(train_capi.Common) == 32
    assert ctypes.sizeof(train_capi.FfnForward) == 32 + 9 * 8 + 6 * 8
    assert ctypes.sizeof(train_capi.FfnBackward) == 32 + 15 * 8 + 7 * 8
    assert ctypes.sizeof(train_capi.LossForward) == 32 + 6 * 8 + 6 * 8 + 8
    assert ctypes.sizeof(train_capi.LossBackward) == 32 + 8 * 8 + 7 * 8 + 8
    assert ctypes.sizeof(train_capi.Orthogonalize) == 32 + 3 * 8 + 6 * 8 + 8 + 16 + 8
    assert train_capi.Orthogonalize.eps.offset == 32 + 9 * 8 + 8 + 16


def test_cpu_tensors_and_wrong_types_are_refused():
    x, w = torch.zeros(4, 8, dtype=torch.float16), torch.zeros(16, 8, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        llm_hgemm.gated_ffn(x, w, w, w.t())
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        llm_hgemm.linear_cross_entropy(x, w, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="g must be a CUDA tensor"):
        llm_hgemm.orthogonalize(w)


def ffn_args(**change):
    p = 1 << 20   # an aligned address that is never read
    a = train_capi.FfnForward(train_capi.Common(), p, p, p, p, p, p, None, None, None, 0, 16, 64, 128, 64, 64)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change", [
    {"tokens": 0}, {"tokens": -1}, {"tokens": 2 ** 31}, {"hidden": 60}, {"inter": 4}, {"out": 0}, {"x": None},
    {"gate": None}, {"y": None}, {"h": (1 << 20) + 8}, {"ldx": 56}, {"ldx": 68}, {"silu": 1 << 20},
    {"common": train_capi.Common(dtype=2)}, {"common": train_capi.Common(splits=17)}, {"common": train_capi.Common(splits=-1)},
    {"common": train_capi.Common(flags=capi.FLAG_OUT_F32)},
], ids=str)
def test_c_abi_refuses_ffn_arguments(change):
    assert train_capi.run("ffn_forward", ffn_args(**change)) == capi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("tile", [1, 32, 96, 320, 0x2000 | 128, 0x1000])
def test_c_abi_refuses_unknown_tiles(tile):
    assert train_capi.run("ffn_forward", ffn_args(common=train_capi.Common(tile=tile))) == capi.ERR_UNKNOWN_CONFIG


@pytest.mark.parametrize("change", [
    {"tokens": 0}, {"vocab": 0}, {"hidden": 12}, {"target": None}, {"lse": None}, {"loss": None}, {"workspace": None},
    {"workspace": (1 << 20) + 4}, {"reduction": 3}, {"reduction": -1}, {"ldx": 8},
], ids=str)
def test_c_abi_refuses_loss_arguments(change):
    p = 1 << 20
    a = train_capi.LossForward(train_capi.Common(), p, p, p, p, p, p, 1 << 30, 4, 16, 100, 16, -100, 0, 0)
    for k, v in change.items():
        setattr(a, k, v)
    assert train_capi.run("loss_forward", a) == capi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("change", [
    {"tokens": 0}, {"dloss": None}, {"dx": (1 << 20) + 2}, {"dweight": (1 << 20) + 2}, {"piece": -1}, {"workspace": None},
], ids=str)
def test_c_abi_refuses_loss_gradient_arguments(change):
    p = 1 << 20
    a = train_capi.LossBackward(train_capi.Common(), p, p, p, p, p, p, p, p, 1 << 30, 4, 16, 100, 16, -100, 0, 0, 0)
    for k, v in change.items():
        setattr(a, k, v)
    assert train_capi.run("loss_backward", a) == capi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("change", [
    {"batch": 0}, {"batch": 65536}, {"rows": 0}, {"cols": -3}, {"steps": -1}, {"ldg": 4}, {"g": None}, {"out": None},
    {"workspace": None}, {"workspace": (1 << 20) + 128}, {"eps": -1.0}, {"eps": float("nan")}, {"batch_stride": -8},
], ids=str)
def test_c_abi_refuses_orthogonalize_arguments(change):
    p = 1 << 20
    a = train_capi.Orthogonalize(train_capi.Common(), p, p, p, 1 << 30, 1, 200, 300, 300, 0, 5, 0, *NEWTON_SCHULZ, 0.0, 1e-7)
    for k, v in change.items():
        setattr(a, k, v)
    assert train_capi.run("orthogonalize", a) == capi.ERR_INVALID_ARGUMENT


def test_null_arguments_and_workspaces():
    lib = train_capi.load()
    for name in ("ffn_forward", "ffn_backward", "loss_forward", "loss_backward", "orthogonalize"):
        assert getattr(lib, f"hgemm_sm100_{name}")(None, None) == capi.ERR_INVALID_ARGUMENT
        assert getattr(lib, f"hgemm_sm100_{name}_workspace")(None) == 0


def test_module_refuses_other_linears():
    a, b = nn.Linear(8, 16, bias=False), nn.Linear(16, 8, bias=False)
    TrainableSwiGLU(a, nn.Linear(8, 16, bias=False), b)
    for parts in ((a, a, nn.Linear(16, 8)), (a, b, b), (a, a, a), (a, a, None)):
        with pytest.raises(ValueError):
            TrainableSwiGLU(*parts)


def test_reference_ffn_matches_autograd():
    torch.manual_seed(0)
    x, g, u, d, dy = (torch.randn(*s).half() for s in ((5, 6), (7, 6), (7, 6), (4, 7), (5, 4)))
    leaves = [t.double().requires_grad_() for t in (x, g, u, d)]
    y = (torch.nn.functional.silu(leaves[0] @ leaves[1].T) * (leaves[0] @ leaves[2].T)) @ leaves[3].T
    for (value, err), want in zip(ref.ffn(x, g, u, d, dy), [y, *torch.autograd.grad(y, leaves, dy.double())]):
        assert torch.allclose(value, want) and bool((err > 0).all())


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_reference_loss_matches_torch(reduction):
    torch.manual_seed(1)
    x, w = torch.randn(6, 5).half(), torch.randn(9, 5).half()
    t = torch.tensor([0, 8, -100, 3, 3, -100])
    dl = torch.rand(6) if reduction == "none" else torch.tensor(3.0)
    a, b = x.double().requires_grad_(), w.double().requires_grad_()
    value = torch.nn.functional.cross_entropy(a @ b.T, t, reduction=reduction)
    grads = torch.autograd.grad(value, [a, b], dl.double())
    for (got, _), want in zip(ref.loss(x, w, t, reduction, -100, dl), [value, *grads]):
        assert torch.allclose(got, want)


def test_reference_orthogonalize_matches_the_steps():
    torch.manual_seed(2)
    g = torch.randn(6, 11).half()
    a, b, c = NEWTON_SCHULZ
    x = g.double() / (torch.linalg.vector_norm(g.double()) + 1e-7)
    for _ in range(5):
        p = x @ x.T
        x = a * x + (b * p + c * (p @ p)) @ x
    value, err = ref.orthogonalize(g, 5, NEWTON_SCHULZ, 1e-7)
    assert torch.allclose(value, x, atol=1e-9) and 0 < err < 1


def test_fingerprint_leaves_the_training_operators_out(tmp_path, monkeypatch):
    """A dispatch table stays valid when only the training operators change."""
    from llm_hgemm import provenance

    names = {rel for rel, _ in provenance._sources()}
    assert not names & provenance._APART
    assert all((provenance.REPO_ROOT / rel).is_file() for rel in provenance._APART)
    assert {"include/hgemm_sm100.h", "llm-tensorcore-hgemm_b200/csrc/hgemm_kernels.cuh",
            "llm-tensorcore-hgemm_b200/csrc/host/bindings.cpp"} <= names


def test_trainable_mlps_keeps_the_parameters():
    from llm_hgemm.integration import trainable_mlps

    class Mlp(nn.Module):
        def __init__(self, act, dtype=torch.float16):
            super().__init__()
            self.gate_proj, self.up_proj = (nn.Linear(8, 16, bias=False, dtype=dtype) for _ in range(2))
            self.down_proj = nn.Linear(16, 8, bias=False, dtype=dtype)
            self.act_fn = act

    model = nn.ModuleDict({"a": Mlp(nn.SiLU()), "b": nn.ModuleList([Mlp(nn.SiLU()), Mlp(nn.GELU())]),
                           "c": Mlp(nn.SiLU(), torch.float32)})
    before = {n: id(p) for n, p in model.named_parameters()}
    assert trainable_mlps(model) == 2
    assert isinstance(model["a"], TrainableSwiGLU) and isinstance(model["b"][0], TrainableSwiGLU)
    assert not isinstance(model["b"][1], TrainableSwiGLU) and not isinstance(model["c"], TrainableSwiGLU)
    assert {n: id(p) for n, p in model.named_parameters()} == before
