"""Which MLPs ``trainable_mlps`` replaces, and which projections its block takes
(CPU): only those that its one operator computes."""

import pytest
import torch
from torch import nn

from llm_hgemm.integration import trainable_mlps
from llm_hgemm.training import TrainableSwiGLU


class Mlp(nn.Module):
    def __init__(self, **parts):
        super().__init__()
        linear = lambda m, n: nn.Linear(m, n, bias=False, dtype=torch.float16)   # noqa: E731
        self.gate_proj, self.up_proj, self.down_proj = linear(8, 16), linear(8, 16), linear(16, 8)
        self.act_fn = nn.SiLU()
        for name, part in parts.items():
            setattr(self, name, part)

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class Doubled(nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


class Renamed(nn.Linear):
    pass


def plain_linear(kind=nn.Linear):
    return kind(8, 16, bias=False, dtype=torch.float16)


def nothing(*args):
    return None


def own_forward(module):
    module.forward = lambda x: x


CHANGES = {
    "subclass": lambda m: setattr(m, "up_proj", plain_linear(Doubled)),
    "own forward": lambda m: own_forward(m.gate_proj),
    "forward hook": lambda m: m.gate_proj.register_forward_hook(nothing),
    "forward pre-hook": lambda m: m.down_proj.register_forward_pre_hook(nothing),
    "backward hook": lambda m: m.up_proj.register_full_backward_hook(nothing),
    "backward pre-hook": lambda m: m.up_proj.register_full_backward_pre_hook(nothing),
    "hook of the MLP": lambda m: m.register_forward_hook(nothing),
    "own forward of the MLP": lambda m: own_forward(m),
    "hook of the activation": lambda m: m.act_fn.register_forward_hook(nothing),
    "dropout": lambda m: setattr(m, "dropout", nn.Dropout(0.1)),
    "parameter": lambda m: setattr(m, "scale", nn.Parameter(torch.ones(1))),
    "buffer": lambda m: m.register_buffer("scale", torch.ones(1)),
}


@pytest.mark.parametrize("change", CHANGES)
def test_an_mlp_that_does_more_stays(change):
    model = nn.ModuleDict({"plain": Mlp(), "other": Mlp()})
    CHANGES[change](model["other"])
    assert trainable_mlps(model) == 1
    assert isinstance(model["plain"], TrainableSwiGLU) and isinstance(model["other"], Mlp)


def test_a_subclass_with_the_same_forward_is_taken():
    model = nn.ModuleDict({"a": Mlp(gate_proj=plain_linear(Renamed))}).eval()
    assert trainable_mlps(model) == 1 and not model["a"].training


@pytest.mark.parametrize("change", [k for k in CHANGES if k in ("subclass", "own forward") or k.endswith("ward hook")
                                    or k.endswith("pre-hook")])
def test_the_block_refuses_projections_that_do_more(change):
    mlp = Mlp()
    block = TrainableSwiGLU(mlp.gate_proj, mlp.up_proj, mlp.down_proj)
    CHANGES[change](mlp)
    with pytest.raises(ValueError, match="hooks or a forward of their own"):
        TrainableSwiGLU(mlp.gate_proj, mlp.up_proj, mlp.down_proj)
    if change != "subclass":     # that one is another module
        with pytest.raises(RuntimeError, match="got hooks"):
            block(torch.zeros(2, 8, dtype=torch.float16))
