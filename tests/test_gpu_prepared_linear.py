"""GPU: weights of a projection that are prepared inside a captured graph."""
import pytest
import torch

from weftmoe_b200.fp8 import fp8_linear, prepare_fp8_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("training", (False, True))
def test_a_captured_preparation_serves_calls_behind_its_replays(training):
    g = torch.Generator("cuda").manual_seed(70)
    weight = torch.randn(300, 256, device="cuda", dtype=torch.bfloat16, generator=g)
    x = torch.randn(40, 256, device="cuda", dtype=torch.bfloat16, generator=g, requires_grad=training)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prepared = prepare_fp8_linear(weight, training=training)
        inside = fp8_linear(x.detach(), weight, prepared)
    for factor in (1.0, -0.5):
        new = torch.randn(300, 256, device="cuda", generator=g).bfloat16() * factor
        weight.data.copy_(new)                                    # by way of .data: the stamp is the captured version's
        graph.replay()
        torch.cuda.synchronize()
        got, want = fp8_linear(x, weight, prepared), fp8_linear(x, new, prepare_fp8_linear(new, training=training))
        assert torch.equal(inside, want) and torch.equal(got, want)
        if training:
            dy = torch.ones_like(got)
            assert torch.equal(*(torch.autograd.grad(y, x, dy)[0] for y in (got, want)))
