"""GPU: the router, the routed experts and a shared expert on the FP8 projection, as one layer of a model calls them,
forward and backward, against the same layer in plain FP32 operations.

Tolerances, as relative 2-norms.  The layer's own kernels round to BF16 between their steps (half a step 2^-8 per value):
3 x 2^-8 for the routed part, the bound the layer's own tests use.  An E4M3 rounding is off by at most 2^-4, evenly spread,
so by r = 2^-4 / sqrt(3) = 0.036 in the mean square, and errors of independent roundings add by their squares:
  gate and up rows     x and W rounded                        sqrt(2) r = 0.051
  u = silu(a) b        |a silu'(a) / silu(a)| <= 2 where u counts, so a's error twice and b's once: sqrt(5) 0.051 = 0.114
  shared output        u and W rounded on top                 sqrt(0.114^2 + 2 r^2) = 0.125 = 2^-3
  d u                  dy and W rounded                       0.051
  d a, d b             d u, and the errors of a and b through silu, silu' and b as above: sqrt(0.051^2 + 0.114^2) = 0.125;
                       and for d a the other factor's error once more: sqrt(0.125^2 + 0.114^2) = 0.169
  dx, dW of gate / up  another two roundings                  sqrt(0.169^2 + 2 r^2) = 0.177 < 2^-2
  dW of down           dy and u rounded, u's error            0.125 < 2^-2
The gradients of x and of the router hold exact parts besides."""
import pytest
import torch

from weftmoe_b200 import SingleRankGroup, TensorRuntime, moe
from weftmoe_b200.fp8 import fp8_linear, poll_fp8_matmul, prepare_fp8_linear
from weftmoe_b200.router import route_and_balance, route_tokens

pytestmark = pytest.mark.gpu

TOKENS, EXPERTS, TOP_K, HIDDEN, INNER = 300, 16, 4, 256, 128


def far(got, want):
    return ((got.double() - want.double()).norm() / want.double().norm()).item()


def plain_layer(x, weights, shared, w1, w2, routes):
    """The same in FP32 operations, with the given routes."""
    gate_up, down = shared
    logits = x @ weights.t()
    gates = logits.gather(1, routes.long()).softmax(1)
    y = torch.zeros_like(x)
    for k in range(TOP_K):
        ab = torch.einsum("th,tih->ti", x, w1[routes[:, k].long()])
        u = torch.nn.functional.silu(ab[:, :INNER]) * ab[:, INNER:]
        y = y + gates[:, k:k + 1] * torch.einsum("ti,thi->th", u, w2[routes[:, k].long()])
    ab = x @ gate_up.t()
    shared_y = (torch.nn.functional.silu(ab[:, :INNER]) * ab[:, INNER:]) @ down.t()
    counts = torch.bincount(routes.flatten().long(), minlength=EXPERTS)
    loss = EXPERTS * (counts / counts.sum() * logits.softmax(1).mean(0)).sum()
    return y, shared_y, loss


@pytest.fixture(scope="module")
def tensors():
    g = torch.Generator("cuda").manual_seed(40)
    make = lambda *shape, scale=1.0: (torch.randn(*shape, device="cuda", generator=g) * scale).bfloat16()
    return {"x": make(TOKENS, HIDDEN), "router": make(EXPERTS, HIDDEN, scale=HIDDEN ** -0.5),
            "w1": make(EXPERTS, 2 * INNER, HIDDEN, scale=HIDDEN ** -0.5),
            "w2": make(EXPERTS, HIDDEN, INNER, scale=INNER ** -0.5),
            "gate_up": make(2 * INNER, HIDDEN, scale=HIDDEN ** -0.5), "down": make(HIDDEN, INNER, scale=INNER ** -0.5),
            "dy": make(TOKENS, HIDDEN)}


def layer(runtime, t, gate_up_q, down_q):
    logits = (t["x"].float() @ t["router"].float().t())
    routes, gates, counts, loss = route_and_balance(logits, TOP_K)
    y = moe(runtime, t["x"], routes, gates, t["w1"], t["w2"])
    ab = fp8_linear(t["x"], t["gate_up"], gate_up_q)
    u = torch.nn.functional.silu(ab[:, :INNER]) * ab[:, INNER:]
    return routes, counts, loss, y, fp8_linear(u, t["down"], down_q)


def test_a_layer_of_router_experts_and_shared_expert(tensors):
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        runtime = TensorRuntime(group=SingleRankGroup(), experts=EXPERTS, top_k=TOP_K, hidden=HIDDEN, intermediate=INNER,
                                max_tokens=TOKENS, max_rows=TOKENS * TOP_K + EXPERTS * 128, training=True,
                                stream=stream)
        t = {k: v.clone().requires_grad_(k != "dy") for k, v in tensors.items()}
        prepared = prepare_fp8_linear(t["gate_up"]), prepare_fp8_linear(t["down"])
        routes, counts, loss, y, shared = layer(runtime, t, *prepared)
        assert counts.sum().item() == TOKENS * TOP_K
        (y.float() * t["dy"]).sum().add((shared.float() * t["dy"]).sum()).add(0.5 * loss).backward()
        got = {k: v.grad for k, v in t.items() if v.grad is not None}
        poll_fp8_matmul()
        runtime.drain()

        w = {k: v.float().requires_grad_(k != "dy") for k, v in tensors.items()}
        plain_y, plain_shared, plain_loss = plain_layer(w["x"], w["router"], (w["gate_up"], w["down"]), w["w1"], w["w2"],
                                                        routes)
        assert far(y, plain_y) < 3 * 2.0 ** -8 and far(shared, plain_shared) < 2.0 ** -3
        assert abs(loss.item() - plain_loss.item()) < 1e-5
        ((plain_y + plain_shared) * w["dy"]).sum().add(0.5 * plain_loss).backward()
        for name in ("w1", "w2"):
            assert far(got[name], w[name].grad) < 3 * 2.0 ** -8, name
        for name in ("x", "router", "gate_up", "down"):
            assert far(got[name], w[name].grad) < 2.0 ** -2, name
        del y, shared, loss, plain_y, plain_shared, plain_loss
        runtime.close()


def test_a_captured_decode_step(tensors):
    """Router, experts and shared projection captured in one graph and replayed on other tokens."""
    tokens = 8
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), torch.no_grad():
        runtime = TensorRuntime(group=SingleRankGroup(), experts=EXPERTS, top_k=TOP_K, hidden=HIDDEN, intermediate=INNER,
                                max_tokens=tokens, max_rows=tokens * TOP_K + EXPERTS * 128, training=False, stream=stream,
                                decode_only=True)
        x = tensors["x"][:tokens].clone()
        routes = torch.empty(tokens, TOP_K, dtype=torch.int32, device="cuda")
        gates = torch.empty(tokens, TOP_K, device="cuda")
        weight = tensors["gate_up"]
        prepared = prepare_fp8_linear(weight, training=False)

        def step():
            r, g = route_tokens(x.float() @ tensors["router"].float().t(), TOP_K)
            routes.copy_(r)
            gates.copy_(g)
            return runtime.inference(0, x, routes, gates, tensors["w1"], tensors["w2"]), fp8_linear(x, weight, prepared)

        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y, ab = step()
        x.copy_(tensors["x"][50:50 + tokens])
        graph.replay()
        got = y.clone(), ab.clone()
        want = step()
        stream.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        del graph
        runtime.close()
