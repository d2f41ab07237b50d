"""GPU: the router operators on finite logits of any magnitude, against their definitions in 64 bits.

Tolerances.  U = 2^-24.  With d the largest difference of a row's logits that counts (beyond 88, exp(-d) is below every
normal FP32 number), an exponential of such a difference is off by 1.3 d U (its argument's rounding, and log2 e's as an
FP32 number, 0.23 U) and 4 U (the exponential itself, 2 units in the last place).  The difference is exact: logits
within a factor of two of each other subtract exactly, and of two others at these magnitudes one vanishes.  Term and sum
each carry that much; the sum adds at most 32 + 5 terms, reciprocal, divisions and products 1 to 2 U each:
REL = (2.6 d + 64) U.  Gradients as in test_gpu_router.py: 6 REL of the terms before they cancel, then the rounding to
the logits' type; the loss 256 U more for sums over rows."""
import math

import pytest
import torch

from tests.router_reference import reference
from tests.test_gpu_router import TYPES, U, close, vector
from weftmoe_b200.router import balance_loss, route_and_balance, route_tokens

pytestmark = pytest.mark.gpu

REL = (2.6 * 88 + 64) * U
EXPERTS, TOP_K = 40, 5
VALUES = [sign * value for value in (2.0 ** 22, 2.0 ** 23 - 0.5, 2.0 ** 23, 2.0 ** 24, 1e8, 5e9, 1e10, 1e20, 9e29, 2e30, 3e38)
          for sign in (1, -1)]


def rows_around(value, dtype):
    """All equal, a few steps apart, beside ordinary logits, beside absent experts, and of both signs."""
    base = torch.tensor(value, dtype=torch.float64).to(TYPES[dtype]).double()
    step = 2.0 ** (math.floor(math.log2(abs(base.item()))) - {"fp32": 23, "bf16": 7}[dtype])
    g = torch.Generator().manual_seed(3)
    x = torch.full((8, EXPERTS), base.item(), dtype=torch.float64)
    x[1] -= math.copysign(step, value) * torch.randint(0, 7, (EXPERTS,), generator=g)
    x[2, ::3] = 0.0
    x[3, 4:] = -math.inf
    x[4] = torch.randn(EXPERTS, generator=g, dtype=torch.float64)
    x[5, 1::2] *= -1
    x[6, 7] -= math.copysign(step, value)
    x[7, :2] = -math.inf
    return x.to(TYPES[dtype])


def gradient_close(got, want, dtype):
    tolerance = 6 * REL * want["reach"] + torch.finfo(dtype).eps / 2 * want["dlogits"].abs() + 1e-37
    close(got, want["dlogits"], tolerance, "dlogits")


@pytest.mark.parametrize("bias", (False, True))
@pytest.mark.parametrize("score, renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                                ("sigmoid", False)])
@pytest.mark.parametrize("dtype", ("fp32", "bf16"))
@pytest.mark.parametrize("value", VALUES)
def test_routes_gates_and_loss(value, dtype, score, renormalize, bias):
    logits, dgates = rows_around(value, dtype), vector(8 * TOP_K, 4).view(8, TOP_K)
    options = dict(score=score, renormalize=renormalize)
    bias = vector(EXPERTS, 5, 0.1) if bias else None
    on_gpu = {**options, "bias": None if bias is None else bias.cuda()}
    want = reference(logits, TOP_K, bias=bias, dgates=dgates, dloss=0.7, **options)
    x = logits.cuda().requires_grad_()
    routes, gates, counts, loss = route_and_balance(x, TOP_K, **on_gpu)
    assert torch.equal(routes.cpu(), want["routes"]) and torch.equal(counts.cpu(), want["counts"])
    close(gates, want["gates"], REL * want["gates"] + 1e-37, "gates")
    close(loss, want["loss"], (REL + 256 * U) * want["loss"], "loss")
    dx, = torch.autograd.grad((gates, loss), x, (dgates.cuda(), torch.tensor(0.7, device="cuda")))
    gradient_close(dx, want, logits.dtype)

    alone = route_tokens(x, TOP_K, **on_gpu)
    assert torch.equal(alone[0], routes) and torch.equal(alone[1], gates)
    dx, = torch.autograd.grad(alone[1], x, dgates.cuda())
    gradient_close(dx, reference(logits, TOP_K, bias=bias, dgates=dgates, **options), logits.dtype)


def test_one_such_row_leaves_the_loss_of_the_others():
    """Rows that a finite mask value fills add equal shares to the loss, not NaN."""
    logits = torch.randn(300, EXPERTS, generator=torch.Generator().manual_seed(6))
    logits[17] = -1e10
    counts = torch.arange(EXPERTS, dtype=torch.int32)
    want = reference(logits, 1, counts=counts, dloss=1.0)
    x = logits.cuda().requires_grad_()
    loss = balance_loss(x, counts.cuda())
    close(loss, want["loss"], (REL + 256 * U) * want["loss"], "loss")
    gradient_close(torch.autograd.grad(loss, x)[0], want, logits.dtype)
