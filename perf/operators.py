"""Cases of the router and dense FP8 operators: what is measured, their plain forms and their definitions in 64 bits.

Five operators, in the order in which a layer uses them:

  route    router logits [T, E] -> routes and gates of the K chosen experts, and the logits' gradient
  balance  per-expert counts of given routes, the balance loss of the logits, and its gradient
  step     both of these in one pass over the logits, forward and backward (a training step of a router)
  matmul   E4M3 matrix product with an FP32 scale for each block of 128
  linear   a projection on such products: BF16 in and out, quantised on the way, with both gradients
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------- cases
def _router(name, kind, tokens, experts, top_k, **more):
    case = {"name": name, "kind": kind, "tokens": tokens, "experts": experts, "top_k": top_k, "score": "softmax",
            "bias": False, "renormalize": True, "scale": 1.0, "dtype": "fp32", "train": True, "padding": 0.0,
            "sequences": 0}
    return {**case, **more}


def _matmul(name, m, n, k, **more):
    case = {"name": name, "kind": "matmul", "m": m, "n": n, "k": k, "a_block_rows": 1, "b_block_rows": 128,
            "out": "bf16", "mantissas": False}
    return {**case, **more}


def _linear(name, tokens, inputs, outputs, **more):
    case = {"name": name, "kind": "linear", "tokens": tokens, "inputs": inputs, "outputs": outputs, "train": True}
    return {**case, **more}


def listed():
    return [
        # one decode step's tokens: nothing but latency
        _router("route decode 64", "route", 64, 256, 6, dtype="bf16", train=False),
        # a prompt through a router that selects by a corrected sigmoid score, padded rows among it; odd length
        _router("route biased sigmoid 4099", "route", 4099, 256, 8, score="sigmoid", bias=True, scale=2.5,
                padding=0.1),
        # the balance loss of one micro-batch whose routes another router chose
        _router("balance 8192x256", "balance", 8192, 256, 8),
        # the same for a packed batch of ragged sequences, some of them empty, with padding; uneven expert count
        _router("balance 13 ragged sequences", "balance", 5003, 160, 6, score="sigmoid", dtype="bf16", padding=0.05,
                sequences=13),
        # a training step of the router: headline layer of this repository's benchmark
        _router("step 8192x256", "step", 8192, 256, 8),
        # the largest router step: long batch, many experts, a loss for each of 16 sequences
        _router("step 65536x512", "step", 65536, 512, 8, score="sigmoid", bias=True, dtype="bf16", sequences=16),
        # a dense projection of 64 decode tokens: the weights are read once
        _matmul("matmul decode 64", 64, 4096, 4096),
        # odd sizes, scales with mantissas as imported checkpoints carry them, FP32 result
        _matmul("matmul odd any scales", 1237, 1000, 1100, mantissas=True, out="fp32"),
        # a prompt's projection, the largest product
        _matmul("matmul 8192x4096x4096", 8192, 4096, 4096),
        # a weight gradient: both operands in 1 x 128 blocks along the tokens, FP32 result
        _matmul("matmul weight gradient", 4096, 2048, 8190, b_block_rows=1, out="fp32"),
        # a projection for one token
        _linear("linear one token", 1, 4096, 2048, train=False),
        # forward and backward of a projection over the headline batch
        _linear("linear training step 8192", 8192, 2048, 4096),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    kind = rng.choice(("route", "balance", "step", "matmul", "linear"))
    if kind == "matmul":
        most = 8192 * 4096 * 4096
        while True:
            m, n, k = _log_uniform(rng, 1, 8192), _log_uniform(rng, 64, 8192), _log_uniform(rng, 64, 8192)
            if m * n * k <= most:
                break
        b_block_rows = rng.choice((128, 128, 1))
        return _matmul("", m, n, k, b_block_rows=b_block_rows, out=rng.choice(("bf16", "fp32")),
                       mantissas=rng.random() < 0.3)
    if kind == "linear":
        most = 8192 * 2048 * 4096
        while True:
            t, i, o = _log_uniform(rng, 1, 8192), _log_uniform(rng, 64, 8192), _log_uniform(rng, 64, 8192)
            if t * i * o <= most:
                break
        return _linear("", t, i, o, train=rng.random() < 0.6)
    experts = _log_uniform(rng, 8, 512)
    tokens = _log_uniform(rng, 1, 65536)
    top_k = rng.randint(1, min(16, experts))
    score = rng.choice(("softmax", "sigmoid"))
    return _router("", kind, tokens, experts, top_k, score=score, bias=kind != "balance" and rng.random() < 0.4,
                   renormalize=rng.random() < 0.7, scale=rng.choice((1.0, 2.5)),
                   dtype=rng.choice(("fp32", "bf16", "fp16")), train=kind != "route" or rng.random() < 0.6,
                   padding=rng.choice((0.0, 0.1)), sequences=0 if kind == "route" else rng.choice((0, 0, 3, 16)))


def work(case):
    """Bytes and operations no implementation can do without: inputs once, outputs once."""
    if case["kind"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // 128)
        scales = 4 * kb * (-(-m // case["a_block_rows"]) + -(-n // case["b_block_rows"]))
        return {"bytes": (m + n) * k + scales + m * n * (2 if case["out"] == "bf16" else 4), "flops": 2 * m * n * k}
    if case["kind"] == "linear":
        t, i, o = case["tokens"], case["inputs"], case["outputs"]
        if not case["train"]:
            return {"bytes": 2 * t * i + i * o + 2 * t * o, "flops": 2 * t * i * o}
        # x, dy, W and W^T once; y, dx and dW once
        return {"bytes": 2 * t * i + 2 * t * o + 2 * i * o + 2 * t * o + 2 * t * i + 2 * i * o, "flops": 6 * t * i * o}
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    size = 4 if case["dtype"] == "fp32" else 2
    kind, rows = case["kind"], max(1, case["sequences"])
    routed = t * k * 4 * (2 if kind != "balance" else 1)                       # routes (and gates)
    moved = t * e * size + routed + (t if case["padding"] else 0)
    if kind != "route":
        moved += rows * e * 4
    if case["train"]:
        moved += t * e * size + (t * k * 4 if kind != "balance" else 0)        # the gradient, and the gates' gradient
    return {"bytes": moved, "flops": t * e * (14 if case["train"] else 6)}


# ---------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "matmul":
        return _prepare_matmul(case, g)
    if case["kind"] == "linear":
        return _prepare_linear(case, g)
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    popular = torch.randn(e, device="cuda", generator=g) * 0.5                 # experts differ in popularity
    logits = (torch.randn(t, e, device="cuda", generator=g) * 1.5 + popular).to(DTYPES[case["dtype"]])
    state = {"case": case, "padding_mask": None, "sequences": None, "bias": None}
    if case["padding"]:
        state["padding_mask"] = torch.rand(t, device="cuda", generator=g) < case["padding"]
        logits = torch.where(state["padding_mask"][:, None], float("nan"), logits)   # what padding holds is no matter
    if case["sequences"]:
        cuts = torch.randint(0, t + 1, (case["sequences"] - 1,), device="cuda", generator=g).sort().values
        cuts[:1] = 0                                                           # at least one empty sequence
        ends = torch.tensor([0, t], device="cuda")
        state["sequences"] = torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)
    if case["bias"]:
        state["bias"] = torch.randn(e, device="cuda", generator=g) * 0.05
    state["logits"] = logits
    if case["kind"] == "balance":
        state["routes"] = torch.rand(t, e, device="cuda", generator=g).topk(k, dim=1).indices.to(torch.int32)
        if case["padding"]:
            state["routes"][state["padding_mask"]] = -1
    if case["train"]:
        state["dgates"] = torch.randn(t, k, device="cuda", generator=g)
    return state


def _codes(rows, columns, g):
    """E4M3 values as a quantiser leaves them: roughly normal, near the type's top in each block; padding zero."""
    padded = -(-columns // 128) * 128
    values = torch.randn(rows, padded, device="cuda", generator=g) * 110
    values[:, columns:] = 0
    return values.clamp_(-448, 448).to(torch.float8_e4m3fn)


def _scales(rows, columns, block_rows, mantissas, g):
    shape = (-(-rows // block_rows), -(-columns // 128))
    scales = torch.exp2(torch.randint(-9, -5, shape, device="cuda", generator=g).float())
    if mantissas:
        scales = scales * (1 + torch.rand(shape, device="cuda", generator=g))
    return scales


def _prepare_matmul(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    state = {"case": case, "a": _codes(m, k, g), "b": _codes(n, k, g),
             "a_scales": _scales(m, k, case["a_block_rows"], case["mantissas"], g),
             "b_scales": _scales(n, k, case["b_block_rows"], case["mantissas"], g)}
    if own:
        from weftmoe_b200.fp8 import FP8Tensor
        state["own_a"] = FP8Tensor(state["a"], state["a_scales"], (m, k), case["a_block_rows"])
        state["own_b"] = FP8Tensor(state["b"], state["b_scales"], (n, k), case["b_block_rows"])
    return state


def _prepare_linear(case, g):
    t, i, o = case["tokens"], case["inputs"], case["outputs"]
    weight = (torch.randn(o, i, device="cuda", generator=g) / math.sqrt(i)).to(torch.bfloat16)
    state = {"case": case, "weight": weight, "x": torch.randn(t, i, device="cuda", generator=g).to(torch.bfloat16)}
    if case["train"]:
        state["dy"] = (torch.randn(t, o, device="cuda", generator=g) * 1e-3).to(torch.bfloat16)
    # both sides keep the weight quantised, as a program does between two optimizer steps
    if own:
        from weftmoe_b200.fp8 import prepare_fp8_linear
        state["prepared"] = prepare_fp8_linear(weight, training=case["train"])
    else:
        state["weight_values"] = _rounded(weight.float(), 128)
    return state


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return {"route": _own_route, "balance": _own_balance, "step": _own_step, "matmul": _own_matmul,
                "linear": _own_linear}[case["kind"]](state, case)
    with torch.no_grad():
        return {"route": _plain_router, "balance": _plain_router, "step": _plain_router, "matmul": _plain_matmul,
                "linear": _plain_linear}[case["kind"]](state, case)


LOSS_WEIGHT = 0.01     # what a training program multiplies the balance loss by


def _own_route(state, case):
    from weftmoe_b200.router import route_tokens
    logits = state["logits"].detach().requires_grad_(case["train"])
    routes, gates = route_tokens(logits, case["top_k"], score=case["score"], renormalize=case["renormalize"],
                                 scale=case["scale"], bias=state["bias"], padding_mask=state["padding_mask"])
    out = {"routes": routes, "gates": gates.detach()}
    if case["train"]:
        out["dlogits"], = torch.autograd.grad(gates, logits, state["dgates"])
    return out


def _own_balance(state, case):
    from weftmoe_b200.router import balance_loss, expert_counts
    logits = state["logits"].detach().requires_grad_()
    counts = expert_counts(state["routes"], case["experts"], sequences=state["sequences"])
    loss = balance_loss(logits, counts, score=case["score"], padding_mask=state["padding_mask"],
                        sequences=state["sequences"])
    dlogits, = torch.autograd.grad(loss, logits)
    return {"counts": counts, "loss": loss.detach(), "dlogits": dlogits}


def _own_step(state, case):
    from weftmoe_b200.router import route_and_balance
    logits = state["logits"].detach().requires_grad_()
    routes, gates, counts, loss = route_and_balance(
        logits, case["top_k"], score=case["score"], renormalize=case["renormalize"], scale=case["scale"],
        bias=state["bias"], padding_mask=state["padding_mask"], sequences=state["sequences"])
    dlogits, = torch.autograd.grad((gates, LOSS_WEIGHT * loss), logits, (state["dgates"], torch.ones_like(loss)))
    return {"routes": routes, "gates": gates.detach(), "counts": counts, "loss": loss.detach(), "dlogits": dlogits}


def _own_matmul(state, case):
    from weftmoe_b200.fp8 import fp8_matmul
    return fp8_matmul(state["own_a"], state["own_b"], dtype=DTYPES[case["out"]])


def _own_linear(state, case):
    from weftmoe_b200.fp8 import fp8_linear
    if not case["train"]:
        with torch.no_grad():
            return {"y": fp8_linear(state["x"], state["weight"], state["prepared"])}
    x, weight = state["x"].detach().requires_grad_(), state["weight"].requires_grad_()
    y = fp8_linear(x, weight, state["prepared"])
    dx, dweight = torch.autograd.grad(y, (x, weight), state["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dweight}


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_scores(x, score):
    """(s, p) of logits in 32 bits: the scores, and the scores as shares of their row (p = s for softmax)."""
    if score == "softmax":
        s = torch.exp(x - x.amax(dim=1, keepdim=True))
        s = s / s.sum(dim=1, keepdim=True)
        return s, s
    s = 1 / (1 + torch.exp(-x))
    return s, s / s.sum(dim=1, keepdim=True)


def _plain_router(state, case):
    kind, t, e, k = case["kind"], case["tokens"], case["experts"], case["top_k"]
    logits = state["logits"]
    live = torch.ones(t, dtype=torch.bool, device=logits.device)
    if state["padding_mask"] is not None:
        live = ~state["padding_mask"]
    x = torch.where(live[:, None], logits.float(), 0.0)
    s, p = _plain_scores(x, case["score"])
    out = {}
    gradient = torch.zeros_like(x)
    if kind == "balance":
        routes = state["routes"].long()
    else:
        order = x                                  # both scores rise with the logit
        if state["bias"] is not None:              # next to a border: scores in 64 bits
            wide, _ = _plain_scores(x.double(), case["score"])
            order = wide + state["bias"].double()
        routes = order.sort(dim=1, descending=True, stable=True).indices[:, :k]
        chosen = s.gather(1, routes)
        share = chosen / chosen.sum(dim=1, keepdim=True)
        gates = case["scale"] * (share if case["renormalize"] else chosen)
        out["gates"] = torch.where(live[:, None], gates, 0.0)
        if case["train"]:
            dgates = state["dgates"] * case["scale"]
            if case["score"] == "softmax":
                weight = share if case["renormalize"] else chosen
                mean = (weight * dgates).sum(dim=1, keepdim=True)
                if not case["renormalize"]:
                    gradient = -s * mean
                    gradient.scatter_add_(1, routes, weight * dgates)
                else:
                    gradient.scatter_(1, routes, weight * (dgates - mean))
            else:
                slope = 1 / (1 + torch.exp(x.gather(1, routes)))        # 1 - s
                if case["renormalize"]:
                    dgates = share * (dgates - (share * dgates).sum(dim=1, keepdim=True))
                else:
                    dgates = chosen * dgates
                gradient.scatter_(1, routes, dgates * slope)
        routes = torch.where(live[:, None], routes, -1)
        out["routes"] = routes.to(torch.int32)
    if kind != "route":
        rows = max(1, case["sequences"])
        owner = torch.zeros(t, dtype=torch.long, device=x.device)
        if state["sequences"] is not None:         # the last sequence that starts at or before the row
            owner = (torch.arange(t, device=x.device)[:, None] >= state["sequences"][None, 1:].long()).sum(dim=1)
        at = owner[:, None] * e + routes
        counts = torch.zeros(rows * e, dtype=torch.int32, device=x.device)
        counts.scatter_add_(0, at.clamp(min=0).flatten(), (routes >= 0).flatten().to(torch.int32))
        counts = counts.view(rows, e)
        p = torch.where(live[:, None], p, 0.0)
        sums = torch.zeros(rows, e, dtype=torch.float64, device=x.device).index_add_(0, owner, p.double())
        tokens = torch.zeros(rows, device=x.device).index_add_(0, owner, live.float())
        present = (tokens > 0).float().sum().clamp(min=1)
        load = e * counts / counts.sum(dim=1, keepdim=True).clamp(min=1)
        weight = load / (tokens.clamp(min=1) * present)[:, None]
        out["loss"] = (weight * sums).sum().float()
        out["counts"] = counts if case["sequences"] else counts[0]
        per_row = weight[owner]
        push = p * (per_row - (p * per_row).sum(dim=1, keepdim=True))
        if case["score"] == "sigmoid":
            push = push / (1 + torch.exp(x))
        gradient = gradient + (LOSS_WEIGHT if kind == "step" else 1.0) * push
    if case["train"]:
        out["dlogits"] = torch.where(live[:, None], gradient, 0.0).to(logits.dtype)
    return out


def _spread(scales, block_rows, rows, columns):
    return scales.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :columns]


def _plain_matmul(state, case):
    m, n, k = case["m"], case["n"], case["k"]
    a = state["a"].float()[:, :k] * _spread(state["a_scales"], case["a_block_rows"], m, k)
    b = state["b"].float()[:, :k] * _spread(state["b_scales"], case["b_block_rows"], n, k)
    return (a @ b.t()).to(DTYPES[case["out"]])


def _rounded(x, block_rows):
    """The values that E4M3 with a power-of-two scale for each [block_rows x 128] block holds of x [M, K]."""
    m, k = x.shape
    rows, columns = -(-m // block_rows) * block_rows, -(-k // 128) * 128
    padded = torch.zeros(rows, columns, device=x.device)
    padded[:m, :k] = x
    blocks = padded.view(rows // block_rows, block_rows, columns // 128, 128)
    top = blocks.abs().amax(dim=(1, 3), keepdim=True)
    mantissa, exponent = torch.frexp(top)          # top / 448 = mantissa / 0.875 * 2^(exponent - 9)
    scale = torch.exp2((exponent - 9 + (mantissa > 0.875)).clamp(min=-126).float())
    scale = torch.where(top == 0, 1.0, scale)
    held = (blocks / scale).to(torch.float8_e4m3fn).float() * scale
    return held.view(rows, columns)[:m, :k]


def _plain_linear(state, case):
    x, w = state["x"].float(), state["weight_values"]
    out = {"y": (_rounded(x, 1) @ w.t()).to(torch.bfloat16)}
    if case["train"]:
        dy = state["dy"].float()
        out["dx"] = (_rounded(dy, 1) @ w).to(torch.bfloat16)
        out["dweight"] = (_rounded(dy.t().contiguous(), 1) @ _rounded(x.t().contiguous(), 1).t()).to(torch.bfloat16)
    return out


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    if case["kind"] == "matmul":
        return _exact_matmul(state, case)
    if case["kind"] == "linear":
        return _exact_linear(state, case)
    return _exact_router(state, case)


def _exact_router(state, case):
    """The definitions, differentiated by autograd: only live rows take part."""
    kind, t, e, k = case["kind"], case["tokens"], case["experts"], case["top_k"]
    device = state["logits"].device
    keep = torch.arange(t, device=device)
    if state["padding_mask"] is not None:
        keep = keep[~state["padding_mask"]]
    x = state["logits"][keep].double().requires_grad_()
    scores = x.softmax(dim=1) if case["score"] == "softmax" else x.sigmoid()
    out, total = {}, x.sum() * 0
    if kind == "balance":
        routes = state["routes"][keep].long()
    else:
        by = scores.detach() + state["bias"].double() if state["bias"] is not None else x.detach()
        routes = torch.argsort(-by, dim=1, stable=True)[:, :k]
        gates = scores.take_along_dim(routes, 1)
        if case["renormalize"]:
            gates = gates / gates.sum(1, keepdim=True)
        gates = gates * case["scale"]
        if case["train"]:
            total = total + (gates * state["dgates"][keep].double()).sum()
        out["gates"] = torch.zeros(t, k, dtype=torch.float64, device=device).index_copy(0, keep, gates.detach())
        out["routes"] = torch.full((t, k), -1, dtype=torch.int32, device=device).index_copy(0, keep, routes.to(torch.int32))
    if kind != "route":
        edges = [0, t] if state["sequences"] is None else state["sequences"].tolist()
        shares = scores / scores.sum(1, keepdim=True)
        counts, losses = [], []
        for first, last in zip(edges[:-1], edges[1:]):
            inside = (keep >= first) & (keep < last)
            chosen = routes[inside]
            counts.append(torch.bincount(chosen.flatten(), minlength=e))
            if chosen.shape[0]:
                load = counts[-1].double() * e / counts[-1].sum()
                losses.append((load * shares[inside].mean(0)).sum())
        loss = torch.stack(losses).mean() if losses else x.sum() * 0
        total = total + loss * (LOSS_WEIGHT if kind == "step" else 1.0)
        counts = torch.stack(counts).to(torch.int32)
        out["counts"] = counts if case["sequences"] else counts[0]
        out["loss"] = loss.detach()
    if case["train"]:
        gradient, = torch.autograd.grad(total, x)
        out["dlogits"] = torch.zeros(t, e, dtype=torch.float64, device=device).index_copy(0, keep, gradient)
    return out


def _exact_matmul(state, case):
    m, n, k = case["m"], case["n"], case["k"]
    rows_a = torch.arange(m, device="cuda") // case["a_block_rows"]
    rows_b = torch.arange(n, device="cuda") // case["b_block_rows"]
    block = torch.arange(k, device="cuda") // 128
    a = state["a"][:, :k].double() * state["a_scales"].double()[rows_a][:, block]
    b = state["b"][:, :k].double() * state["b_scales"].double()[rows_b][:, block]
    return torch.einsum("mk,nk->mn", a, b)


def _exact_held(x, block_rows):
    """E4M3 by its definition: 3 bits behind the leading one down to 2^-6, steps of 2^-9 below; ties to even."""
    x = x.double()
    m, k = x.shape
    row, column = torch.arange(m, device=x.device) // block_rows, torch.arange(k, device=x.device) // 128
    tops = torch.zeros(int(row[-1]) + 1, k, dtype=torch.float64, device=x.device)
    tops = tops.index_reduce(0, row, x.abs(), "amax")
    tops = torch.zeros(tops.shape[0], int(column[-1]) + 1, dtype=torch.float64, device=x.device).index_reduce(
        1, column, tops, "amax")
    power = torch.ceil(torch.log2(torch.where(tops > 0, tops, 448.0) / 448)).clamp(min=-126)
    scale = torch.exp2(power)[row][:, column]
    y = x / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale


def _exact_linear(state, case):
    x = state["x"]
    w = _exact_held(state["weight"], 128)
    out = {"y": torch.einsum("ti,oi->to", _exact_held(x, 1), w)}
    if case["train"]:
        dy = state["dy"]
        out["dx"] = torch.einsum("to,oi->ti", _exact_held(dy, 1), w)
        out["dweight"] = torch.einsum("ot,it->oi", _exact_held(dy.t(), 1), _exact_held(x.t(), 1))
    return out
