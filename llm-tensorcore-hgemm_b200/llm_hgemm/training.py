"""Training operators on the library's tensor-core core: the gated feed-forward
block, the loss of a language-model head and the orthogonalised update of a
weight, each with hand-written sm_100a kernels (no reference counterpart: the
reference, llm_hgemm/integration.py:8-46, is inference-only).

They take FP16 or BF16 CUDA tensors and weights in ``nn.Linear``'s layout
(``[out_features, in_features]``), which are read on every call: nothing is
packed or kept, so an optimizer may change them between calls. A weight without
gaps between its rows, with 16-byte aligned rows and sizes that are multiples of
8, is read where it is; any other (a slice of columns, say) is copied in each
forward and each backward pass. Sums are FP32. Launches
go to the current stream of the tensors' device; scratch comes from torch's
caching allocator, so calls on different streams and captured graphs do not
share any. A backward pass can be captured into a CUDA graph, together with its forward
pass or after it (``torch.cuda.make_graphed_callables``); it is refused while an
eager graph of the same tensors from the default stream lives (delete the eager
call's outputs first). Like the rest of the package there is no CPU or library fallback.
"""

from __future__ import annotations

import torch
from torch import nn

from . import _C
from .capi import status_string

#: Coefficients of the quintic Newton-Schulz step of the Muon optimizer.
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)


def gated_ffn(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor) -> torch.Tensor:
    """SwiGLU block ``(silu(x @ gate.T) * (x @ up.T)) @ down.T``, differentiable in
    all four tensors.

    ``x`` is ``[..., H]`` (any strides), ``gate`` and ``up`` ``[I, H]``, ``down``
    ``[O, I]``; the result is ``[..., O]``. Two launches: gate and up are one
    product whose epilogue writes the gated activation, then the down
    projection. Where a gradient is wanted the gated activation and its two
    derivatives are kept (``3 * tokens * I`` elements); the backward pass is two
    launches more, one whose epilogue turns the activation's gradient into
    those of the pre-activations, and one for all wanted gradients together.
    Where the sums of the result or of ``x``'s gradient come in parts (few
    tokens, a nearly empty last wave), one more launch adds them, each way. H, I and O that are no multiples of 8 work through padded copies.
    Gradients of gradients and forward mode are refused.
    """
    return _C.gated_ffn(x, gate, up, down)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *,
                         reduction: str = "mean", ignore_index: int = -100) -> torch.Tensor:
    """``cross_entropy(x @ weight.T, target)`` without the logits, in FP32,
    differentiable in ``x`` and ``weight``.

    ``x`` is ``[..., H]``, ``weight`` ``[V, H]``, ``target`` ``[...]`` (int64 or
    int32). ``reduction``: ``"none"`` (shape of ``target``), ``"mean"`` over the
    targets that are not ``ignore_index`` (NaN when there is none) or
    ``"sum"``. Ignored targets have loss 0 and gradient 0, and add
    nothing to the weight's, whatever ``x`` holds there. A target outside
    ``[0, V)`` that is not ``ignore_index`` gives that token a NaN loss (and NaN
    gradients) instead of a device assertion. The forward pass keeps one number
    per token; the backward pass forms the logits again, a piece of the
    vocabulary at a time. Gradients of gradients and forward mode are refused.
    """
    return _C.linear_cross_entropy(x, weight, target, reduction, ignore_index)


def orthogonalize(g: torch.Tensor, *, steps: int = 5,
                  coefficients: tuple[float, float, float] = NEWTON_SCHULZ,
                  eps: float = 1e-7) -> torch.Tensor:
    """The last two dimensions of ``g`` with all singular values moved towards 1
    (the update direction of the Muon optimizer): ``X = g / (norm(g) + eps)``,
    then ``steps`` times ``X = a X + (b A + c A A) X`` with ``A = X X^T`` (of the
    shorter side).

    Leading dimensions are a batch of matrices, each normalised by itself. A
    zero matrix gives zeros. The steps run on FP16 elements (scaled by a power
    of two) whatever the dtype of ``g``, so no element may pass 255 on the way, or
    65504 in ``A`` and the polynomial: coefficients that keep the singular values
    near 1 stay far below. No gradient is recorded.
    """
    a, b, c = coefficients
    return _C.orthogonalize(g, steps, a, b, c, eps)


def check_status() -> None:
    """Waits for the current device and raises ``RuntimeError`` if a kernel of an
    operator above gave up: every wait inside the kernels has a time limit, after
    which they return with their results incomplete. Each call of an operator
    raises it as well, for those of earlier calls that have run by then, so this is
    for the end of a run and for replayed graphs. Raising clears it."""
    torch.cuda.synchronize()
    status = _C.training_status(True)
    if status != 0:
        raise RuntimeError(f"a kernel of the training operators failed ({status_string(status)}); its results are not valid")


def runs_as_is(module: nn.Module) -> bool:
    """Whether calling ``module`` is its class's ``forward`` and nothing else: no
    hooks, no ``forward`` or ``__call__`` of its own."""
    return not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks
                or module._backward_pre_hooks or "forward" in vars(module)
                or type(module).__call__ is not nn.Module.__call__)


def is_plain_linear(module) -> bool:
    """Whether calling ``module`` multiplies by its weight and nothing else, so that
    an operator may read the weight instead: no bias, no subclass with another
    ``forward`` (quantisation, adapters), no hooks."""
    return (isinstance(module, nn.Linear) and module.bias is None and type(module).forward is nn.Linear.forward
            and runs_as_is(module))


class TrainableSwiGLU(nn.Module):
    """SwiGLU MLP that trains through :func:`gated_ffn`; the counterpart of the
    inference-only ``HgemmSwiGLU``. It holds the projections it is built from
    as ``gate_proj``, ``up_proj`` and ``down_proj``, so parameters, state dict
    and optimizers stay as they are. The projections' weights are used, they are
    not called: ones with another ``forward`` or with hooks are refused, also
    where these came after the block was built. Under ``torch.autocast`` the
    input and the weights are cast to its type, as ``nn.Linear`` does."""

    def __init__(self, gate: nn.Linear, up: nn.Linear, down: nn.Linear):
        super().__init__()
        if not all(is_plain_linear(lin) for lin in (gate, up, down)):
            raise ValueError("requires bias-free nn.Linear projections without hooks or a forward of their own")
        if gate.weight.shape != up.weight.shape or down.in_features != gate.out_features:
            raise ValueError("gate/up/down shapes do not form an MLP")
        self.gate_proj, self.up_proj, self.down_proj = gate, up, down

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        for lin in (self.gate_proj, self.up_proj, self.down_proj):
            if not is_plain_linear(lin):
                raise RuntimeError("a projection got hooks, a bias or another forward, which this block does not run")
        weights = (self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight)
        if torch.is_autocast_enabled("cuda"):     # what the projections' F.linear does there
            dtype = torch.get_autocast_dtype("cuda")
            x, *weights = (t.to(dtype) for t in (x, *weights))
        return gated_ffn(x, *weights)
