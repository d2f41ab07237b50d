"""Derivatives that the operators do not have are refused before anything runs, not left out without a word: on the CPU
through the binding, which refuses before it looks at the device, and on the GPU through the public calls."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from weftmoe_b200 import _lib, fp8
from weftmoe_b200.fp8 import fp8_linear, fp8_matmul, prepare_fp8_linear, quantize_fp8
from weftmoe_b200.router import balance_loss, expert_counts, route_and_balance, route_tokens


def dual(*shape, dtype=torch.float32, device="cpu", requires_grad=False):
    primal = torch.zeros(*shape, dtype=dtype, device=device).requires_grad_(requires_grad)
    return forward_ad.make_dual(primal, torch.ones(*shape, dtype=dtype, device=device))


@pytest.mark.parametrize("requires_grad", (False, True))
def test_forward_mode_is_refused(requires_grad):
    binding = _lib.binding()
    counts, plain = torch.zeros(8, dtype=torch.int32), torch.zeros(4, 8)
    empty = torch.empty(0)
    with forward_ad.dual_level():
        x = dual(4, 8, requires_grad=requires_grad)
        for call in (lambda: binding.route(x, 2, 0, True, 1.0, None, None, None, False),
                     lambda: binding.route(x, 2, 0, True, 1.0, None, None, None, True),
                     lambda: binding.balance(x, counts, 0, None, None),
                     lambda: binding.fp8_linear(x, plain, empty, empty, None, None),
                     lambda: binding.fp8_linear(plain, x, empty, empty, None, None)):
            with pytest.raises(RuntimeError, match="forward mode"):
                call()


@pytest.mark.gpu
def test_forward_mode_is_refused_by_the_public_calls():
    counts = torch.ones(8, dtype=torch.int32, device="cuda")
    weight = torch.randn(64, 128, device="cuda", dtype=torch.bfloat16)
    prepared = prepare_fp8_linear(weight)
    with forward_ad.dual_level():
        x = dual(4, 8, device="cuda")
        for call in (lambda: route_tokens(x, 2), lambda: route_and_balance(x, 2), lambda: balance_loss(x, counts),
                     lambda: fp8_linear(dual(4, 128, dtype=torch.bfloat16, device="cuda"), weight, prepared)):
            with pytest.raises(RuntimeError, match="forward mode"):
                call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward mode"):
            route_tokens(x, 2)
        routes, gates = route_tokens(forward_ad.unpack_dual(x).primal, 2)     # without its tangent it is an input
        assert expert_counts(routes, 8).sum().item() == 8
    route_tokens(x, 2)                                                        # behind the level there is no tangent


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x = torch.randn(6, 16, device="cuda", requires_grad=True)
    weight = torch.randn(64, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = torch.randn(6, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    counts = torch.ones(16, dtype=torch.int32, device="cuda")
    for value, leaf in ((route_tokens(x, 2)[1].sum(), x), (balance_loss(x, counts), x),
                        (route_and_balance(x, 2)[3], x), (fp8_linear(y, weight, prepare_fp8_linear(weight)).sum(), y)):
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad(value, leaf, create_graph=True)


def outs_with_history(device):
    leaf = torch.zeros(8, 16, device=device, requires_grad=True)
    return leaf, leaf * 2, leaf[:, :], (torch.zeros(8, 32, device=device, requires_grad=True) + 1)[:, 8:24]


@pytest.mark.parametrize("accumulate", (False, True))
def test_an_out_with_a_gradient_is_refused(accumulate):
    a, b = (fp8._allocate((rows, 256), 1, torch.empty(0)) for rows in (8, 16))
    for out in outs_with_history("cpu"):
        before = out._version
        with pytest.raises(RuntimeError, match="requires a gradient"):
            fp8_matmul(a, b, dtype=torch.float32, out=out, accumulate=accumulate)
        assert out._version == before
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
        fp8_matmul(a, b, dtype=torch.float32, out=dual(8, 16))


@pytest.mark.gpu
def test_an_out_without_a_gradient_is_taken():
    a, b = (quantize_fp8(torch.randn(rows, 256, device="cuda", dtype=torch.bfloat16)) for rows in (8, 16))
    want = fp8_matmul(a, b, dtype=torch.float32)
    for out in outs_with_history("cuda"):
        with pytest.raises(RuntimeError, match="requires a gradient"):
            fp8_matmul(a, b, dtype=torch.float32, out=out)
        with torch.no_grad():                                     # the caller's own part, as for torch's calls
            assert torch.equal(fp8_matmul(a, b, dtype=torch.float32, out=out), want)
    leaf = torch.zeros(8, 16, device="cuda", requires_grad=True)
    leaf.grad = torch.ones(8, 16, device="cuda")
    fp8_matmul(a, b, dtype=torch.float32, out=leaf.grad, accumulate=True)
    assert torch.equal(leaf.grad, want + 1)
