"""GPU: the balance loss's gradient where the load is nearly even, as a well-trained router has it.  Its slope by a
token's shares is f - 1 up to a constant, here down to 1e-8 of f; tolerances are those of test_gpu_router.py, relative to
f - 1 and not to f."""
import pytest
import torch

from tests.router_reference import reference
from tests.test_gpu_router import U, close, gradient_close, make, rel
from weftmoe_b200.router import balance_loss

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences", (None, (0, 30, 30, 64)))
@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
@pytest.mark.parametrize("load, apart", [(1000, 1), (1000000, 3), (100000000, 1), (2000000000, 50)])
def test_gradient_of_a_nearly_even_load(load, apart, score, sequences):
    logits, experts = make(64, 40), 40
    rows = 1 if sequences is None else len(sequences) - 1
    counts = load + torch.randint(-apart, apart + 1, (rows, experts), generator=torch.Generator().manual_seed(90))
    counts = (counts[0] if sequences is None else counts).int()
    offsets = None if sequences is None else torch.tensor(sequences, dtype=torch.int32)
    want = reference(logits, 1, score=score, counts=counts, dloss=3.0, sequences=offsets)
    x = logits.cuda().requires_grad_()
    loss = balance_loss(x, counts.cuda(), score=score, sequences=None if offsets is None else offsets.cuda())
    close(loss, want["loss"], (rel(logits) + 256 * U) * want["loss"], "loss")
    gradient_close(torch.autograd.grad(3.0 * loss, x)[0], want, logits)
