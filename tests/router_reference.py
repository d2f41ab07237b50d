"""The router operators' definitions in 64 bits (include/weftmoe_b200.h, wm_router), row by row where that is
plainest.  Gradients come from autograd on these definitions."""
import torch


def live_rows(tokens, padding_mask=None, sequences=None):
    live = torch.ones(tokens, dtype=torch.bool)
    if padding_mask is not None:
        live &= ~padding_mask.cpu().bool()
    if sequences is not None:
        offsets = sequences.tolist()
        at = torch.arange(tokens)
        live &= (at >= offsets[0]) & (at < offsets[-1])
    return live


def scores_of(x, score):
    """x float64 [T, E]; rows need an available expert."""
    return x.softmax(1) if score == "softmax" else x.sigmoid()


def choose(x, top_k, score="softmax", bias=None):
    """Routes of float64 logits, one row at a time; -1 behind the last available expert."""
    routes = torch.full((x.shape[0], top_k), -1, dtype=torch.int32)
    for t in range(x.shape[0]):
        available = [e for e in range(x.shape[1]) if x[t, e] > float("-inf")]
        if not available:
            continue
        by = x[t]
        if bias is not None:
            by = scores_of(x[t:t + 1], score)[0] + bias.double().cpu()
        by = by.tolist()
        order = sorted(available, key=lambda e: (-by[e], e))[:top_k]
        routes[t, :len(order)] = torch.tensor(order, dtype=torch.int32)
    return routes


def shares(x, score):
    """s / sum of the row; for rows of very negative sigmoids the sum is taken in the logarithm."""
    if score == "softmax":
        return x.softmax(1)
    return torch.nn.functional.logsigmoid(x).softmax(1)


def gates_of(x, routes, score, renormalize, scale):
    """Gates of rows that have a route (float64, differentiable); -1 gives 0."""
    held = routes.long().clamp(min=0)
    there = routes >= 0
    if renormalize:
        picked = x.gather(1, held)
        if score == "sigmoid":
            picked = torch.nn.functional.logsigmoid(picked)
        picked = picked.masked_fill(~there, float("-inf"))
        gates = picked.softmax(1)
    else:
        gates = scores_of(x, score).gather(1, held)
    return scale * torch.where(there, gates, 0.0)


def reference(logits, top_k, *, score="softmax", renormalize=True, scale=1.0, bias=None, padding_mask=None,
              sequences=None, counts=None, routes=None, dgates=None, dloss=None):
    """dict of routes, gates, counts, loss and dlogits (of sum(gates * dgates) + dloss * loss); reach [T, E] bounds
    what the terms of dlogits add up to before they cancel: every element is a weight times differences of factors,
    reach is that weight times the largest factor of its row."""
    tokens, experts = logits.shape
    live = live_rows(tokens, padding_mask, sequences)
    wide = logits.detach().cpu().double()
    usable = live & (wide.masked_fill(~live[:, None], 0.0) > float("-inf")).any(1)
    at = usable.nonzero()[:, 0]
    x = wide[at].clone().requires_grad_()
    out = {"routes": torch.full((tokens, top_k), -1, dtype=torch.int32),
           "gates": torch.zeros(tokens, top_k, dtype=torch.float64),
           "dlogits": torch.zeros(tokens, experts, dtype=torch.float64),
           "reach": torch.zeros(tokens, experts, dtype=torch.float64)}
    picked = choose(x.detach(), top_k, score, bias) if routes is None else routes.cpu()[at]
    out["routes"][at] = picked
    total = torch.zeros((), dtype=torch.float64)
    if at.numel():
        gates = gates_of(x, picked, score, renormalize, scale)
        out["gates"][at] = gates.detach()
        if dgates is not None:
            total = total + (gates * dgates.cpu().double()[at]).sum()
            weight = torch.zeros_like(x)
            if not renormalize and score == "softmax":
                weight = scale * scores_of(x.detach(), score)
            held = torch.where(picked >= 0, gates.detach(), 0.0)
            weight = weight.scatter_add(1, picked.long().clamp(min=0), held)
            out["reach"][at] += weight * dgates.cpu().double()[at].abs().amax(1, keepdim=True)
    offsets = [0, tokens] if sequences is None else sequences.tolist()
    own_counts = torch.zeros(len(offsets) - 1, experts, dtype=torch.int32)
    losses = []
    for b, (first, last) in enumerate(zip(offsets[:-1], offsets[1:])):
        inside = (at >= first) & (at < last)
        chosen = picked[inside].flatten()
        own_counts[b] = torch.bincount(chosen[chosen >= 0].long(), minlength=experts)
        if inside.any():
            c = (own_counts if counts is None else counts.cpu().view(-1, experts))[b].double()
            load = experts * c / c.sum().clamp(min=1)
            losses.append((load * shares(x[inside], score).mean(0)).sum())
            if dloss is not None:
                p = shares(x[inside].detach(), score)
                out["reach"][at[inside]] += abs(dloss) * p * (load - 1).abs().max() / inside.sum()
    loss = torch.stack(losses).mean() if losses else torch.zeros((), dtype=torch.float64)
    out["counts"] = own_counts if sequences is not None else own_counts[0]
    out["loss"] = loss.detach()
    if dloss is not None:
        total = total + dloss * loss
    if total.requires_grad:
        gradient, = torch.autograd.grad(total, x)
        out["dlogits"][at] = gradient
    return out
