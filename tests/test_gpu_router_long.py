"""GPU: the balance loss of batches so long that a warp adds the shares of several hundred rows one after another.

Tolerance, with U = 2^-24: a share is within (2 |x|max + 64) U as in test_gpu_router.py; the sums add at most
ceil(tokens / (1184 blocks x 8 warps)) rows one after another, then 8 warps, ceil(records / 32) records and 32 sums, all of
one sign and U each."""
import pytest
import torch

from tests.test_gpu_router import U, close, rel
from weftmoe_b200.router import balance_loss, expert_counts, route_and_balance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
@pytest.mark.parametrize("tokens, experts", [(3000001, 16), (10000000, 4), (2 ** 26 - 1, 2)])
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


def test_as_many_sequences_as_there_may_be():
    """65535 sequences of 0 to 5 tokens: routes, counts, the loss (its mean over live sequences) and the gradient."""
    sequences, experts, top_k = 65535, 8, 2
    g = torch.Generator("cuda").manual_seed(81)
    lengths = torch.randint(0, 6, (sequences,), device="cuda", generator=g)
    offsets = torch.nn.functional.pad(lengths.cumsum(0), (1, 0)).int()
    tokens = offsets[-1].item() + 3                               # the last three belong to no sequence
    logits = torch.randn(tokens, experts, device="cuda", generator=g).requires_grad_()
    routes, gates, counts, loss = route_and_balance(logits, top_k, sequences=offsets)
    assert (routes[-3:] == -1).all() and not gates[-3:].any()
    owner = torch.repeat_interleave(torch.arange(sequences, device="cuda"), lengths)
    held = routes[:-3].long()
    own = torch.zeros(sequences, experts, dtype=torch.int64, device="cuda")
    own.index_put_((owner[:, None].expand_as(held), held), torch.ones_like(held), accumulate=True)
    assert torch.equal(counts.long(), own) and torch.equal(expert_counts(routes, experts, sequences=offsets), counts)

    wide = logits.detach()[:-3].double()
    shares = wide.softmax(1)
    live = lengths > 0
    load = experts * own.double() / own.sum(1, keepdim=True).clamp(min=1)
    mean = torch.zeros(sequences, experts, dtype=torch.float64, device="cuda").index_add_(0, owner, shares)
    mean /= lengths.clamp(min=1)[:, None]
    want = (load * mean).sum(1)[live].mean()
    close(loss, want.cpu(), (rel(logits.detach()) + 256 * U) * want.cpu(), "loss")
    dx, = torch.autograd.grad(loss, logits)
    weight = shares / lengths[owner, None] / live.sum()
    slope = load[owner] - 1
    want = weight * (slope - (shares * slope).sum(1, keepdim=True))
    reach = weight * slope.abs().amax(1, keepdim=True)
    assert not dx[-3:].any()
    assert ((dx[:-3].double() - want).abs() - 6 * rel(logits.detach()) * reach - U * want.abs()).max().item() <= 1e-37
