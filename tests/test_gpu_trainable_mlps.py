"""``TrainableSwiGLU`` where the MLP that it replaces ran (GPU)."""

import pytest
import torch
from torch import nn

from llm_hgemm.training import TrainableSwiGLU
from tests import training_reference as ref
from tests.gpu_helpers import require_cuda
from tests.test_gpu_training import ffn_inputs, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    require_cuda()


def block_of(*weights):
    linears = []
    for w in weights:
        linears.append(nn.Linear(w.shape[1], w.shape[0], bias=False, device="cuda", dtype=w.dtype))
        linears[-1].weight = nn.Parameter(w)
    return TrainableSwiGLU(*linears)


@pytest.mark.parametrize("autocast", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("weight", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("given", [torch.float16, torch.float32], ids=str)
def test_autocast(autocast, weight, given):
    """Inputs and weights of other types, as behind an FP32 norm: the values are
    those of the casts, the gradients come in the types of the leaves."""
    x, gate, up, down, dy = ffn_inputs(35, 64, 136, 72, torch.float32)
    x = x.to(given).requires_grad_()
    block = block_of(*(w.to(weight) for w in (gate, up, down)))
    leaves = [x, block.gate_proj.weight, block.up_proj.weight, block.down_proj.weight]
    dy = dy.to(autocast)
    with torch.autocast("cuda", dtype=autocast):
        y = block(x)
    assert y.dtype == autocast
    want = ref.ffn(*(t.detach().to(autocast) for t in leaves), dy)
    within(y.detach(), want[0])
    for t, got, (value, err) in zip(leaves, torch.autograd.grad(y, leaves, dy), want[1:]):
        assert got.dtype == t.dtype
        # The gradient in the autocast type once more in the leaf's.
        within(got, (value, err + ref.unit(t.dtype) * (value.abs() + err) + ref.floor_of(t.dtype)))


def test_autocast_switched_off_inside():
    x, gate, up, down, _ = ffn_inputs(5, 64, 128, 64, torch.float16)
    block = block_of(gate, up, down)
    want = block(x)
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.autocast("cuda", enabled=False):
        assert torch.equal(block(x), want)
