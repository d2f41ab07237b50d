"""GPU: what a captured backward pass may find behind it.  A leaf's gradient is accumulated on the stream of the graph that
first took it; the legacy default stream cannot join a capture, so gradients that would go there are refused."""
import pytest
import torch

from weftmoe_b200.fp8 import fp8_linear, prepare_fp8_linear
from weftmoe_b200.router import balance_loss, route_and_balance, route_tokens

pytestmark = pytest.mark.gpu
NAMES = ("route", "step", "balance", "linear", "linear, x alone")


def cases():
    logits = torch.randn(64, 32, device="cuda", requires_grad=True)
    counts = torch.ones(32, dtype=torch.int32, device="cuda")
    x = torch.randn(40, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    weight = torch.randn(96, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    prepared = prepare_fp8_linear(weight)
    frozen = weight.detach().clone()
    prepared_frozen = prepare_fp8_linear(frozen)
    return {"route": (lambda: route_tokens(logits, 4)[1], (logits,)),
            "step": (lambda: route_and_balance(logits, 4)[3], (logits,)),
            "balance": (lambda: balance_loss(logits, counts), (logits,)),
            "linear": (lambda: fp8_linear(x, weight, prepared), (x, weight)),
            "linear, x alone": (lambda: fp8_linear(x, frozen, prepared_frozen), (x,))}


@pytest.mark.parametrize("name", NAMES)
def test_gradients_of_a_live_eager_graph_are_refused_in_a_capture(name):
    forward, leaves = cases()[name]
    alive = forward()
    want = torch.autograd.grad(alive, leaves, torch.ones_like(alive), retain_graph=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = forward()                                             # a forward pass alone is no trouble
        with pytest.raises(RuntimeError, match="cannot be captured"):
            torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            y.backward(torch.ones_like(y))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, alive) and all(leaf.grad is None for leaf in leaves)
    del graph, alive, y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = forward()
        got = torch.autograd.grad(y, leaves, torch.ones_like(y))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_that_do_not_go_there_are_captured():
    """The weight is a leaf of a live eager graph, but the captured gradient is the input's alone."""
    g = torch.Generator("cuda").manual_seed(95)
    weight = torch.randn(96, 256, device="cuda", dtype=torch.bfloat16, generator=g, requires_grad=True)
    prepared = prepare_fp8_linear(weight)
    x = torch.randn(40, 256, device="cuda", dtype=torch.bfloat16, generator=g)
    alive = fp8_linear(x, weight, prepared)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = x.clone().requires_grad_()
        y = fp8_linear(inside, weight, prepared)
        dx, = torch.autograd.grad(y, inside, torch.ones_like(y))
    graph.replay()
    torch.cuda.synchronize()
    outside = x.clone().requires_grad_()
    assert torch.equal(y, alive)
    assert torch.equal(dx, torch.autograd.grad(fp8_linear(outside, weight, prepared), outside, torch.ones_like(y))[0])


@pytest.mark.parametrize("name", NAMES)
def test_eager_backward_passes_beside_other_streams_are_as_before(name):
    forward, leaves = cases()[name]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = forward()
        there = torch.autograd.grad(alive, leaves, torch.ones_like(alive), retain_graph=True)
    torch.cuda.current_stream().wait_stream(side)
    here = forward()
    assert torch.equal(alive, here)
    got = torch.autograd.grad(here, leaves, torch.ones_like(here))
    assert all(torch.equal(a, b) for a, b in zip(got, there))
