"""GPU: the balance loss of batches so long that a warp adds the shares of several hundred rows one after another.

Tolerance, with U = 2^-24: a share is within (2 |x|max + 64) U as in test_gpu_router.py; the sums add at most
ceil(tokens / (1184 blocks x 8 warps)) rows one after another, then 8 warps, ceil(records / 32) records and 32 sums, all of
one sign and U each."""
import pytest
import torch

from tests.test_gpu_router import U, close, rel
from weftmoe_b200.router import balance_loss, expert_counts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
@pytest.mark.parametrize("tokens, experts", [(3000001, 16), (10000000, 4)])
def test_loss_of_millions_of_tokens(tokens, experts, score):
    g = torch.Generator("cuda").manual_seed(80)
    logits = torch.randn(tokens, experts, device="cuda", generator=g).clamp(-4, 4)
    logits[:, 1] += 2
    logits.requires_grad_()
    routes = torch.randint(0, experts, (tokens, 2), device="cuda", generator=g, dtype=torch.int32)
    counts = expert_counts(routes, experts)
    assert torch.equal(counts.long(), torch.bincount(routes.flatten().long(), minlength=experts))
    loss = balance_loss(logits, counts, score=score)
    dx, = torch.autograd.grad(loss, logits)

    wide = logits.detach().double()
    scores = wide.softmax(1) if score == "softmax" else wide.sigmoid()
    shares = scores / scores.sum(1, keepdim=True)
    load = experts * counts.double() / counts.sum().double()
    want = (load * shares.mean(0)).sum()
    added = -(-tokens // (1184 * 8)) + 8 + 38 + 32
    close(loss, want.cpu(), (rel(logits.detach()) + added * U) * want.cpu(), "loss")
    slope = shares / tokens * ((load - 1) - (shares * (load - 1)).sum(1, keepdim=True))
    if score == "sigmoid":
        slope *= 1 - scores
    reach = shares / tokens * (load - 1).abs().max()
    off = (dx.double() - slope).abs() - 6 * rel(logits.detach()) * reach - U * slope.abs()
    assert off.max().item() <= 1e-37
