"""Backward passes captured into CUDA graphs the ways that torch's own modules
allow (GPU)."""

import copy

import pytest
import torch
from torch import nn

import llm_hgemm
from llm_hgemm.training import TrainableSwiGLU
from tests.gpu_helpers import require_cuda
from tests.test_gpu_training import loss_inputs, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    require_cuda()


def block():
    torch.manual_seed(0)
    sizes = ((64, 136), (64, 136), (136, 64))
    return TrainableSwiGLU(*(nn.Linear(a, b, bias=False) for a, b in sizes)).to("cuda", torch.bfloat16)


def test_graphed_callables():
    """torch keeps the warm-up's outputs, on a stream of their own, during the capture."""
    b, x = block(), normal(1, 33, 64, dtype=torch.bfloat16)
    leaf = x.clone().requires_grad_()
    y = b(leaf)
    y.float().sum().backward()
    want = [y.detach(), leaf.grad, *(p.grad for p in b.parameters())]
    other = copy.deepcopy(b)
    other.zero_grad()
    del y
    graphed = torch.cuda.make_graphed_callables(other, (x.clone().requires_grad_(),))
    leaf = x.clone().requires_grad_()
    y = graphed(leaf)
    y.float().sum().backward()
    for got, v in zip([y.detach(), leaf.grad, *(p.grad for p in other.parameters())], want):
        assert torch.equal(got, v)


@pytest.mark.parametrize("what", ["ffn", "loss"])
def test_beside_an_eager_graph_of_another_stream(what):
    b, x = block(), normal(1, 33, 64, dtype=torch.bfloat16).requires_grad_()
    _, w, t = loss_inputs(33, 64, 501, torch.bfloat16)
    w.requires_grad_()
    leaves = [x, w] if what == "loss" else [x, *b.parameters()]
    call = (lambda: llm_hgemm.linear_cross_entropy(x, w, t)) if what == "loss" else (lambda: b(x).float().sum())
    want = torch.autograd.grad(call(), leaves)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        alive = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(call(), leaves)
    for v in out:
        v.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for got, again, v in zip(out, torch.autograd.grad(alive, leaves), want):
        assert torch.equal(got, v) and torch.equal(again, v)


def test_beside_an_eager_graph_of_a_tensor_without_a_wanted_gradient():
    b, x = block(), normal(1, 33, 64, dtype=torch.bfloat16).requires_grad_()
    weights = list(b.parameters())
    want = torch.autograd.grad(b(x).float().sum(), weights)
    alive = x * 2          # on the default stream
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(b(x).float().sum(), weights)
    graph.replay()
    torch.cuda.synchronize()
    for got, v in zip(out, want):
        assert torch.equal(got, v)
    del alive
