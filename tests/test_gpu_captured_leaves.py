"""GPU: what a capture may find of its leaves.  A leaf's gradient is accumulated on the stream of the graph that first
took it; the legacy default stream cannot join a capture, so a forward pass that would lead there is refused."""
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
def test_a_leaf_of_a_live_eager_graph_is_refused_in_a_capture(name):
    forward, leaves = cases()[name]
    alive = forward()
    want = torch.autograd.grad(alive, leaves, torch.ones_like(alive), retain_graph=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device="cuda")
        with pytest.raises(RuntimeError, match="eager graph"):
            forward()
        with torch.no_grad():
            forward()                                             # nothing accumulates behind this
    del graph, alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = forward()
        got = torch.autograd.grad(y, leaves, torch.ones_like(y))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", NAMES)
def test_other_live_graphs_are_no_reason(name):
    """Eager calls beside each other, and a live graph of a side stream, which could join."""
    forward, leaves = cases()[name]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = forward()
    torch.cuda.current_stream().wait_stream(side)
    again = forward()
    assert torch.equal(alive, again)
    del again
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = forward()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(inside, alive)
