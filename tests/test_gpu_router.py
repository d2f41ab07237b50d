"""GPU: the router operators against their definitions in 64 bits.

Tolerances.  U = 2^-24 is half an FP32 step.  An exponential of a difference d is off by |d| U (the subtraction),
4 U (expf, 2 units in the last place); the sums of a row add at most 32 + 5 terms of one sign, divisions and
products 1 U each: a score or gate is within REL = (2 |x|max + 64) U of its value.  A gradient element is a weight
times a difference of two factors, each of the two within 3 REL of `reach` (its weight times its row's largest
factor), so within 6 REL reach; then it is rounded to the logits' type (half a step of it; FP16 has subnormal steps of
2^-24).  Sums over rows add at most 256 more terms one after another (8 warps' rows, then records): 256 U."""
import pytest
import torch

from tests.router_reference import reference
from weftmoe_b200.router import balance_loss, expert_counts, route_and_balance, route_tokens

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def rel(logits):
    finite = logits[torch.isfinite(logits)].float()
    return (2 * (finite.abs().max().item() if finite.numel() else 0.0) + 64) * U


def make(tokens, experts, dtype="fp32", seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed + 1000 * tokens + experts)
    return (torch.randn(tokens, experts, generator=g) * spread).clamp(-12, 12).to(TYPES[dtype])


def vector(length, seed, spread=1.0):
    return torch.randn(length, generator=torch.Generator().manual_seed(seed)) * spread


def close(got, want, tolerance, what):
    got, want = got.detach().cpu().double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    off = (got - want).abs()
    worst = (off - tolerance).nan_to_num(-1).max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: off by {off.nan_to_num(0).max().item():.3e}, {worst:.3e} over the tolerance"


def gradient_close(got, want, logits, factor=1.0):
    tolerance = 6 * factor * rel(logits) * want["reach"] + torch.finfo(logits.dtype).eps / 2 * want["dlogits"].abs()
    if logits.dtype == torch.float16:
        tolerance = tolerance + 2.0 ** -25
    assert got.dtype == logits.dtype and got.shape == want["dlogits"].shape
    close(got, want["dlogits"], tolerance + 1e-37, "dlogits")


def check_route(logits, top_k, dgates=None, bias=None, padding_mask=None, **options):
    want = reference(logits, top_k, dgates=dgates, bias=bias, padding_mask=padding_mask, **options)
    x = logits.cuda().requires_grad_()
    routes, gates = route_tokens(x, top_k, bias=None if bias is None else bias.cuda(),
                                 padding_mask=None if padding_mask is None else padding_mask.cuda(), **options)
    assert routes.dtype == torch.int32 and gates.dtype == torch.float32 and not routes.requires_grad
    assert torch.equal(routes.cpu(), want["routes"])
    close(gates, want["gates"], rel(logits) * want["gates"] + 1e-37, "gates")
    if dgates is not None:
        got, = torch.autograd.grad(gates, x, dgates.cuda())
        gradient_close(got, want, logits)
    with torch.no_grad():
        again = route_tokens(x, top_k, bias=None if bias is None else bias.cuda(),
                             padding_mask=None if padding_mask is None else padding_mask.cuda(), **options)
    assert torch.equal(again[0], routes) and torch.equal(again[1], gates)


@pytest.mark.parametrize("renormalize", (True, False))
@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
@pytest.mark.parametrize("tokens, experts, top_k", [
    (1, 1, 1), (1, 8, 8), (7, 31, 3), (8, 32, 32), (9, 33, 6), (65, 64, 1), (33, 100, 8), (17, 160, 6), (70, 256, 8),
    (5, 257, 17), (13, 512, 32), (6, 600, 5), (3, 1024, 8)])
def test_sizes(tokens, experts, top_k, score, renormalize):
    check_route(make(tokens, experts), top_k, torch.randn(tokens, top_k), score=score, renormalize=renormalize,
                scale=2.5)


@pytest.mark.parametrize("dtype", ("bf16", "fp16"))
@pytest.mark.parametrize("score, renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                                ("sigmoid", False)])
def test_types(dtype, score, renormalize):
    check_route(make(41, 128, dtype), 8, vector(41 * 8, 1).view(41, 8), score=score, renormalize=renormalize)


@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
@pytest.mark.parametrize("experts", (8, 160, 512))
@pytest.mark.parametrize("spread", (0.0, 1e-3, 0.1))
def test_bias_selects_but_does_not_weigh(score, experts, spread):
    check_route(make(37, experts), 6, vector(37 * 6, 2).view(37, 6), score=score, bias=vector(experts, 3, spread))


@pytest.mark.parametrize("value", (torch.finfo(torch.float32).min, -1e10, torch.finfo(torch.float32).max))
@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
@pytest.mark.parametrize("experts, left", [(8, 2), (8, 5), (31, 3), (64, 4), (300, 6)])
def test_bias_of_the_lowest_value_puts_experts_last(experts, left, score, value):
    """All but `left` experts are banned (or, by the largest value, put first); top_k reaches into the others, and two
    that are left are closer than 32 bits tell."""
    bias = torch.full((experts,), value)
    keep = torch.arange(left) * (experts // left)
    bias[keep] = 0.0
    logits = make(21, experts, seed=17)
    logits[:, keep[1]] = logits[:, keep[0]] * (1 + 2 ** -22)
    logits[3, keep] = -float("inf")                              # none of them left
    logits[4, experts // 2:] = -float("inf")
    for top_k in (left, min(left + 2, experts)):
        check_route(logits, top_k, vector(21 * top_k, 18).view(21, top_k), bias=bias, score=score)


@pytest.mark.parametrize("bias", (None, torch.zeros(64)))
def test_ties_go_to_the_lowest_expert(bias):
    logits = torch.randint(-2, 3, (50, 64), generator=torch.Generator().manual_seed(4)).float()
    logits[3] = 0.0
    logits[4, ::2] = -0.0
    check_route(logits, 9, vector(50 * 9, 5).view(50, 9), bias=bias)


def test_scores_that_32_bits_cannot_tell_apart():
    """Neighbouring FP32 logits whose sigmoids are the same FP32 number: the choice goes by the true order, also
    against the index, and a bias of one FP32 step decides where it is larger than their difference."""
    base = torch.full((1, 8), 9.0)
    step = 2.0 ** -20
    base[0] += torch.arange(8) * step
    assert base.float().sigmoid().unique().numel() < 8
    check_route(base, 4, score="sigmoid", bias=torch.zeros(8))
    check_route(base, 4, score="sigmoid", bias=torch.tensor([2.0 ** -24, 0, 0, 0, 0, 0, 2.0 ** -25, 0]))


def test_masks():
    lowest = torch.finfo(torch.float32).min
    logits = make(12, 40)
    logits[0] = float("-inf")                       # nothing is left
    logits[1, 3:] = float("-inf")                   # fewer than top_k
    logits[2, 1:] = float("-inf")
    logits[3, 5:] = lowest                          # finite: available with a vanishing score
    logits[4] = lowest
    logits[5, :20] = float("-inf")
    dgates = vector(12 * 6, 6).view(12, 6)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            want = reference(logits[[0, 1, 2, 5, 6, 7]], 6, score=score, renormalize=renormalize,
                             dgates=dgates[[0, 1, 2, 5, 6, 7]])
            x = logits.cuda().requires_grad_()
            routes, gates = route_tokens(x, 6, score=score, renormalize=renormalize)
            dx, = torch.autograd.grad(gates, x, dgates.cuda())
            at = [0, 1, 2, 5, 6, 7]
            assert torch.equal(routes.cpu()[at], want["routes"])
            close(gates[at], want["gates"], rel(make(12, 40)) * want["gates"] + 1e-37, "gates")
            close(dx[at], want["dlogits"], 6 * rel(make(12, 40)) * want["reach"] + 1e-37, "dlogits")
            assert not torch.isnan(gates).any() and not torch.isnan(dx).any()
            assert routes[3].tolist() == sorted(range(5), key=lambda e: -logits[3, e].item()) + [5]
            assert routes[4].tolist() == [0, 1, 2, 3, 4, 5]
            if score == "softmax" and renormalize:   # six equal logits
                close(gates[4], torch.full((6,), 1 / 6), 8 * U, "equal shares")


@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
def test_padding_rows_hold_anything(score):
    logits, dgates = make(30, 24), vector(30 * 4, 7).view(30, 4)
    mask = torch.zeros(30, dtype=torch.bool)
    mask[::4] = True
    dirty = logits.clone()
    dirty[::8] = float("nan")
    dirty[4::8] = float("inf")
    check_route(logits, 4, dgates, padding_mask=mask, score=score)
    for kind in (torch.bool, torch.uint8):
        x = dirty.cuda().requires_grad_()
        routes, gates = route_tokens(x, 4, padding_mask=mask.to(kind).cuda(), score=score)
        clean = route_tokens(logits.cuda(), 4, padding_mask=mask.cuda(), score=score)
        assert torch.equal(routes, clean[0]) and torch.equal(gates, clean[1])
        dx, = torch.autograd.grad(gates, x, dgates.cuda())
        assert not dx[mask.cuda()].any() and not torch.isnan(dx).any()


@pytest.mark.parametrize("bias", (None, torch.zeros(16)))
def test_rows_without_a_distribution_show(bias):
    logits = make(6, 16)
    logits[1, 5] = float("nan")
    logits[3, 2] = float("inf")
    x = logits.cuda().requires_grad_()
    routes, gates = route_tokens(x, 4, bias=None if bias is None else bias.cuda())
    dx, = torch.autograd.grad(gates.sum(), x)
    assert routes[1].tolist() == routes[3].tolist() == [0, 1, 2, 3]
    assert torch.isnan(gates[[1, 3]]).all() and torch.isnan(dx[[1, 3]]).all()
    assert not torch.isnan(gates[[0, 2, 4, 5]]).any() and not torch.isnan(dx[[0, 2, 4, 5]]).any()


def test_far_logits_keep_their_shares():
    """Sigmoids of -200 are zero in 32 bits; their shares are not.  Softmax of +-80 neither overflows nor loses the top."""
    logits = torch.tensor([[-200.0, -201.0, -202.0, -250.0], [300.0, 299.0, -300.0, 0.0], [-90.0, 80.0, 79.0, 0.0]])
    dgates = torch.tensor([[1.0, -2.0, 0.5]] * 3)
    for score in ("softmax", "sigmoid"):
        check_route(logits, 3, dgates, score=score)
        x = logits.cuda().requires_grad_()
        counts = torch.tensor([5, 1, 0, 3], dtype=torch.int32)
        want = reference(logits, 1, score=score, counts=counts, dloss=2.0)
        loss = balance_loss(x, counts.cuda(), score=score)
        close(loss, want["loss"], (rel(logits) + 256 * U) * want["loss"], "loss")
        dx, = torch.autograd.grad(2.0 * loss, x)
        gradient_close(dx, want, logits)


def test_layouts_other_than_plain_rows():
    wide = make(20, 64)
    dgates = vector(20 * 4, 8).view(20, 4)
    for view in (lambda w: w[:, 16:48], lambda w: w[::2], lambda w: w.t(), lambda w: w[:1].expand(20, 64),
                 lambda w: w.flip(1)):
        leaf = wide.clone().cuda().requires_grad_()
        x = view(leaf)
        routes, gates = route_tokens(x, 4)
        want = reference(view(wide), 4, dgates=dgates[:1].expand(x.shape[0], 4))
        assert torch.equal(routes.cpu(), want["routes"])
        got, = torch.autograd.grad(gates, x, dgates[:1].cuda().expand(x.shape[0], 4))   # an expanded gradient
        gradient_close(got, want, wide)
    leaf = wide.clone().cuda().requires_grad_()
    gates = route_tokens(leaf[:1].expand(20, 64), 4)[1]
    gates.backward(dgates.cuda())
    want = reference(wide[:1].expand(20, 64), 4, dgates=dgates)
    close(leaf.grad[0], want["dlogits"].sum(0), 20 * 6 * rel(wide) * want["reach"].amax(0) + 1e-37, "summed gradient")
    assert not leaf.grad[1:].any()


def test_no_tokens():
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    routes, gates = route_tokens(x, 4)
    assert routes.shape == gates.shape == (0, 4)
    routes, gates, counts, loss = route_and_balance(x, 4)
    assert loss.item() == 0 and not counts.any()
    dx, = torch.autograd.grad(gates.sum() + loss, x)
    assert dx.shape == (0, 16)
    assert not expert_counts(routes, 16).any()


# ------------------------------------------------------------------ counts and loss
OFFSETS = {
    "one": [0, 300], "halves": [0, 150, 300], "empty ones": [0, 0, 7, 7, 7, 130, 300, 300],
    "behind the last": [0, 100, 250], "before the first": [20, 100, 300], "past the end": [0, 200, 400],
    "single rows": list(range(0, 301)),
}


def check_balance(logits, top_k, dgates, dloss, score, dtype="fp32", padding_mask=None, sequences=None, **options):
    seq = None if sequences is None else torch.tensor(sequences, dtype=torch.int32)
    want = reference(logits, top_k, score=score, dgates=dgates, dloss=dloss, padding_mask=padding_mask, sequences=seq,
                     **options)
    on = lambda t: None if t is None else t.cuda()
    x = logits.cuda().requires_grad_()
    options = {k: on(v) if isinstance(v, torch.Tensor) else v for k, v in options.items()}
    routes, gates, counts, loss = route_and_balance(x, top_k, score=score, padding_mask=on(padding_mask),
                                                    sequences=on(seq), **options)
    assert torch.equal(routes.cpu(), want["routes"]) and torch.equal(counts.cpu(), want["counts"])
    assert counts.dtype == torch.int32 and loss.dtype == torch.float32 and loss.ndim == 0
    close(gates, want["gates"], rel(logits) * want["gates"] + 1e-37, "gates")
    close(loss, want["loss"], (rel(logits) + 256 * U) * want["loss"], "loss")
    got, = torch.autograd.grad((gates, loss), x, (dgates.cuda(), torch.tensor(dloss, device="cuda")),
                               retain_graph=True)
    gradient_close(got, want, logits)
    # the two parts alone, and the operators one by one
    part, = torch.autograd.grad(gates, x, dgates.cuda(), retain_graph=True)
    gradient_close(part, reference(logits, top_k, score=score, dgates=dgates, padding_mask=padding_mask, sequences=seq,
                                   **{k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in options.items()}),
                   logits)
    assert torch.equal(expert_counts(routes, logits.shape[1], sequences=on(seq)), counts)
    y = logits.cuda().requires_grad_()
    alone = balance_loss(y, counts, score=score, padding_mask=on(padding_mask), sequences=on(seq))
    assert torch.equal(alone, loss)
    separate, = torch.autograd.grad(alone, y, torch.tensor(dloss, device="cuda"))
    together, = torch.autograd.grad(loss, x, torch.tensor(dloss, device="cuda"))
    assert torch.equal(separate, together)


@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
@pytest.mark.parametrize("offsets", list(OFFSETS))
def test_loss_of_sequences(score, offsets):
    logits = make(300, 40)
    logits[::7, 3] = float("-inf")
    logits[11] = float("-inf")
    mask = torch.zeros(300, dtype=torch.bool)
    mask[5:60:3] = True
    mask[200:215] = True
    check_balance(logits, 5, vector(1500, 9).view(300, 5), 0.3, score, padding_mask=mask, sequences=OFFSETS[offsets])


@pytest.mark.parametrize("score, renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                                ("sigmoid", False)])
@pytest.mark.parametrize("tokens, experts, dtype", [(1, 8, "fp32"), (9, 1, "fp32"), (333, 256, "bf16"),
                                                    (77, 1024, "fp32"), (4000, 64, "fp16"), (1200, 512, "fp32")])
def test_loss_sizes(tokens, experts, dtype, score, renormalize):
    top_k = min(8, experts)
    check_balance(make(tokens, experts, dtype), top_k, vector(tokens * top_k, 10).view(tokens, top_k), -1.5, score,
                  renormalize=renormalize, scale=2.0, bias=vector(experts, 11, 0.1))


def test_everything_is_padding():
    logits = make(10, 8)
    logits[:] = float("nan")
    mask = torch.ones(10, dtype=torch.bool).cuda()
    x = logits.cuda().requires_grad_()
    routes, gates, counts, loss = route_and_balance(x, 2, padding_mask=mask)
    dx, = torch.autograd.grad(gates.sum() + loss, x)
    assert loss.item() == 0 and not counts.any() and (routes == -1).all() and not dx.any()


def test_counts_summed_over_ranks():
    """The loss takes counts as they are given: those of the whole job, or none at all."""
    logits = make(64, 16)
    for counts in (torch.arange(16, dtype=torch.int32) * 100000000, torch.zeros(16, dtype=torch.int32)):
        counts = counts.clamp(max=2 ** 31 - 1)
        want = reference(logits, 2, counts=counts, dloss=1.0)
        x = logits.cuda().requires_grad_()
        loss = balance_loss(x, counts.cuda())
        dx, = torch.autograd.grad(loss, x)
        close(loss, want["loss"], (rel(logits) + 256 * U) * want["loss"], "loss")
        gradient_close(dx, want, logits)


def test_counts_ignore_ids_that_are_no_expert():
    routes = torch.tensor([[0, -1], [7, 8], [2 ** 31 - 1, -2 ** 31], [3, 3]], dtype=torch.int32).cuda()
    assert expert_counts(routes, 8).tolist() == [1, 0, 0, 2, 0, 0, 0, 1]


def test_even_load_gives_one():
    x = torch.zeros(32, 16, device="cuda")
    assert abs(balance_loss(x, torch.full((16,), 4, dtype=torch.int32, device="cuda")).item() - 1) <= 64 * U


def test_gradient_against_differences():
    """Central differences of the operator's own outputs in a random direction v, step h: the third derivative of
    gates and loss is below 8 |v|^3 per element here, so the quotient is off by 8 h^2 n / 6, plus the outputs'
    rounding (REL per term over 2 h)."""
    h, n = 2.0 ** -7, 24 * 4
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            logits, dgates = make(24, 32).cuda(), vector(n, 12).view(24, 4).cuda()
            v = vector(24 * 32, 13).view(24, 32).clamp(-1, 1).cuda()

            def value(x):
                routes, gates, _, _ = route_and_balance(x, 4, score=score, renormalize=renormalize)
                loss = balance_loss(x, counts, score=score)
                return routes, (gates.double() * dgates).sum() + 3 * loss.double()

            counts = torch.randint(0, 50, (32,), dtype=torch.int32, device="cuda",
                                   generator=torch.Generator("cuda").manual_seed(14))
            x = logits.clone().requires_grad_()
            routes, total = value(x)
            slope = (torch.autograd.grad(total, x)[0].double() * v).sum()
            keep = torch.ones(24, dtype=torch.bool, device="cuda")
            for sign in (-1, 1):                      # rows whose choice changes have no derivative
                keep &= (value(logits + sign * h * v)[0] == routes).all(1)
            v = v * keep[:, None]
            slope = (torch.autograd.grad(value(x)[1], x)[0].double() * v).sum()
            quotient = (value(logits + h * v)[1] - value(logits - h * v)[1]) / (2 * h)
            size = dgates.abs().sum().item() + 3 * 32
            assert abs((quotient - slope).item()) <= 8 * h * h / 6 * size + rel(logits) * size / h


def test_same_bits_every_time():
    x = make(5000, 256).cuda().requires_grad_()
    seen = None
    for _ in range(3):
        routes, gates, counts, loss = route_and_balance(x, 8)
        dx, = torch.autograd.grad(gates.sum() + loss, x)
        now = (routes, gates.detach(), counts, loss.detach(), dx)
        assert seen is None or all(torch.equal(a, b) for a, b in zip(seen, now))
        seen = now


def test_captured_forward_and_backward_replay_on_new_inputs():
    first, second = make(200, 64, seed=1).cuda(), make(200, 64, seed=2).cuda()
    static = first.clone().requires_grad_()
    dgates = vector(800, 15).view(200, 4).cuda()

    def step(x):
        routes, gates, counts, loss = route_and_balance(x, 4)
        dx, = torch.autograd.grad((gates, loss), x, (dgates, torch.ones_like(loss)))
        return routes, gates.detach(), counts, loss.detach(), dx

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step(static))
    for data in (first, second):
        with torch.no_grad():
            static.copy_(data)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step(data.clone().requires_grad_())
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_another_stream():
    want = route_and_balance(make(500, 128).cuda(), 6)
    side = torch.cuda.Stream()
    x = make(500, 128).cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = route_and_balance(x, 6)
    del x
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_long_batches_pass_32_bits():
    """4.2 M rows of 512: element offsets beyond 2^31."""
    rows, experts = 4200000, 512
    x = torch.zeros(rows, experts, dtype=torch.bfloat16, device="cuda")
    tail = make(64, experts, "bf16")
    x[-64:] = tail.cuda()
    x.requires_grad_()
    routes, gates, counts, loss = route_and_balance(x, 2)
    want = reference(tail, 2)
    assert torch.equal(routes[-64:].cpu(), want["routes"])
    assert torch.equal(routes[:1000].cpu(), torch.tensor([[0, 1]], dtype=torch.int32).expand(1000, 2))
    assert counts.sum().item() == 2 * rows
    dgates = torch.zeros_like(gates)
    dgates[-64:, 0] = 1.0
    dx, = torch.autograd.grad(gates, x, dgates)
    want = reference(tail, 2, dgates=dgates[-64:].cpu())
    gradient_close(dx[-64:], want, tail)
    assert not dx[:1000].any()


@pytest.mark.parametrize("sequences", (1, 32, 33, 500))
def test_counts_of_no_tokens(sequences):
    routes = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    offsets = torch.zeros(sequences + 1, dtype=torch.int32, device="cuda")
    counts = expert_counts(routes, 5, sequences=offsets)
    assert counts.shape == (sequences, 5) and not counts.any()


@pytest.mark.parametrize("score, bias", [("softmax", None), ("sigmoid", "zeros"), ("sigmoid", "spread"), ("softmax", "spread")])
@pytest.mark.parametrize("experts", (33, 64, 300, 512, 1024))
@pytest.mark.parametrize("top_k", (12, 13, 16, 25, 32))
def test_many_choices(top_k, experts, score, bias):
    """More candidates than lanes: plain rows, rows of few distinct values, rows with masked experts, and rows whose
    values around the border are closer than 32-bit scores tell."""
    logits = make(40, experts, seed=23)
    logits[8:16] = (logits[8:16] * 2).round() / 2
    logits[16] = 0.0
    logits[17] = logits[17].sign()
    logits[18, top_k + 1:] = -float("inf")                      # one expert more than choices
    logits[19, top_k - 2:] = -float("inf")                      # fewer than choices
    logits[24:32] = 0.25 + torch.arange(experts) * 2.0 ** -24   # neighbours one step apart
    logits[28:32] = logits[28:32].flip(1)
    biases = {None: None, "zeros": torch.zeros(experts), "spread": vector(experts, 24, 0.05)}
    check_route(logits, top_k, bias=biases[bias], score=score)
    low = torch.full((2, experts), torch.finfo(torch.float32).min)   # apart: it widens the tolerance of the gates
    low[0, ::3] = 1.0
    check_route(low, top_k, bias=biases[bias], score=score)
