"""Router operators in front of `TensorRuntime` / `moe`: top-k routes with gates, per-expert counts, balance loss.

    routes, gates = route_tokens(logits, top_k)                        # what forward / moe take
    counts = expert_counts(routes, experts)                            # int32 load of each expert
    loss = balance_loss(logits, counts)                                # routes of this or of another router
    routes, gates, counts, loss = route_and_balance(logits, top_k)     # all of it in one pass over the logits

The reference leaves the router to its host framework (weftmoe/megatron.py:164-188 takes routes and gates from it);
the definitions are in include/weftmoe_b200.h beside `wm_router`.  All arithmetic runs in libweftmoe_b200.so; this
file checks arguments, allocates results and joins the calls to autograd.  Every call enqueues on the current
stream of the logits' device, synchronises nothing and may be captured in a CUDA graph; capture a backward pass
together with its forward pass (autograd runs a backward pass on the stream of its forward pass).
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
_SCORES = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS = 1024
MAX_TOP_K = 32
MAX_SEQUENCES = 65535


def _check_logits(logits):
    if not isinstance(logits, torch.Tensor) or logits.ndim != 2 or logits.dtype not in _DTYPES:
        raise ValueError("logits must be a BF16, FP32 or FP16 tensor [tokens, experts]")
    if not 1 <= logits.shape[1] <= MAX_EXPERTS:
        raise ValueError(f"logits must have 1 to {MAX_EXPERTS} experts")


def _check_vector(tensor, what, dtypes, length, like):
    if tensor is None:
        return
    if (not isinstance(tensor, torch.Tensor) or tensor.dtype not in dtypes or tensor.ndim != 1
            or (length is not None and tensor.shape[0] != length)):
        names = " or ".join(str(d).replace("torch.", "") for d in dtypes)
        raise ValueError(f"{what} must be a {names} vector" + (f" of {length}" if length is not None else ""))
    if tensor.device != like.device or not tensor.is_contiguous():
        raise ValueError(f"{what} must be contiguous, on the device of the logits or routes")


def _check_sequences(sequences, like):
    _check_vector(sequences, "sequences", (torch.int32,), None, like)
    if sequences is not None and not 2 <= sequences.shape[0] <= MAX_SEQUENCES + 1:
        raise ValueError(f"sequences must hold the offsets of 1 to {MAX_SEQUENCES} sequences")


def _check_score(score):
    if score not in _SCORES:
        raise ValueError("score must be 'softmax' or 'sigmoid'")


def _check_choice(logits, top_k, scale):
    if not isinstance(top_k, int) or isinstance(top_k, bool) or not 1 <= top_k <= min(MAX_TOP_K, logits.shape[1]):
        raise ValueError(f"top_k must be in [1, min({MAX_TOP_K}, experts)]")
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError("scale must be finite and positive")


def _require_device(tensor, what):
    if not tensor.is_cuda:
        raise ValueError(f"{what} must be on a CUDA device")


def _stream(*tensors):
    """The current stream; it keeps the storage of tensors that were made on another one."""
    stream = torch.cuda.current_stream()
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return stream.cuda_stream


def _rows(logits):
    """The logits as rows of unit column stride (copied only if they are not)."""
    tokens, experts = logits.shape
    plain = (experts == 1 or logits.stride(1) == 1) and (tokens <= 1 or logits.stride(0) >= experts)
    return logits if plain else logits.contiguous()


def _describe(logits, top_k, score, renormalize, scale, bias, padding_mask, sequences):
    tokens, experts = logits.shape
    return _lib.WmRouter(
        logits.data_ptr(), logits.stride(0) if tokens > 1 else experts, _DTYPES[logits.dtype], tokens, experts, top_k,
        _SCORES[score], int(renormalize), scale, 0 if sequences is None else sequences.shape[0] - 1,
        None if bias is None else bias.data_ptr(), None if padding_mask is None else padding_mask.data_ptr(),
        None if sequences is None else sequences.data_ptr())


def _loss_buffers(router, device):
    """(loss, table, workspace) of a call that computes the loss."""
    size = ctypes.c_int64()
    _lib.check(_lib.load().wm_router_workspace(ctypes.byref(router), ctypes.byref(size)))
    return (torch.empty((), dtype=torch.float32, device=device),
            torch.empty(max(1, router.num_sequences) * router.experts + 1, dtype=torch.float32, device=device),
            torch.empty(size.value, dtype=torch.uint8, device=device))


def _backward(logits, router_args, routes, dgates, table, dloss):
    with torch.cuda.device(logits.device):
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        router = _describe(logits, *router_args)
        _lib.check(_lib.load().wm_router_backward(
            ctypes.byref(router), _lib.ptr(routes), _lib.ptr(dgates), _lib.ptr(table), _lib.ptr(dloss),
            _lib.ptr(dlogits), _stream(logits, *router_args[-2:], routes, dgates, table, dloss)))
    return dlogits


def _route(logits, top_k, score, renormalize, scale, bias, padding_mask, sequences, balance):
    """(routes, gates, counts, loss, table); the last three are None without the loss."""
    device = logits.device
    with torch.cuda.device(device):
        routes = torch.empty((logits.shape[0], top_k), dtype=torch.int32, device=device)
        gates = torch.empty((logits.shape[0], top_k), dtype=torch.float32, device=device)
        router = _describe(logits, top_k, score, renormalize, scale, bias, padding_mask, sequences)
        counts = loss = table = workspace = None
        if balance:
            loss, table, workspace = _loss_buffers(router, device)
            shape = (logits.shape[1],) if sequences is None else (sequences.shape[0] - 1, logits.shape[1])
            counts = torch.empty(shape, dtype=torch.int32, device=device)
        _lib.check(_lib.load().wm_router_forward(
            ctypes.byref(router), _lib.ptr(routes), _lib.ptr(gates), _lib.ptr(counts), _lib.ptr(loss),
            _lib.ptr(table), _lib.ptr(workspace), 0 if workspace is None else workspace.numel(),
            _stream(logits, bias, padding_mask, sequences)))
    return routes, gates, counts, loss, table


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, score, renormalize, scale, bias, padding_mask):
        rows = _rows(logits)
        routes, gates, *_ = _route(rows, top_k, score, renormalize, scale, bias, padding_mask, None, False)
        ctx.options = (top_k, score, renormalize, scale)
        ctx.save_for_backward(rows, routes, padding_mask)
        ctx.mark_non_differentiable(routes)
        return routes, gates

    @staticmethod
    @once_differentiable
    def backward(ctx, _, dgates):
        rows, routes, padding_mask = ctx.saved_tensors
        dlogits = _backward(rows, (*ctx.options, None, padding_mask, None), routes,
                            dgates.float().contiguous(), None, None)
        return (dlogits, *[None] * 6)


class _RouteAndBalance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, score, renormalize, scale, bias, padding_mask, sequences):
        rows = _rows(logits)
        routes, gates, counts, loss, table = _route(rows, top_k, score, renormalize, scale, bias, padding_mask,
                                                    sequences, True)
        ctx.options = (top_k, score, renormalize, scale)
        ctx.save_for_backward(rows, routes, padding_mask, sequences, table)
        ctx.mark_non_differentiable(routes, counts)
        ctx.set_materialize_grads(False)
        return routes, gates, counts, loss

    @staticmethod
    @once_differentiable
    def backward(ctx, _routes, dgates, _counts, dloss):
        rows, routes, padding_mask, sequences, table = ctx.saved_tensors
        if dgates is None and dloss is None:
            return (None,) * 8
        if dgates is None:
            routes = None
        else:
            dgates = dgates.float().contiguous()
        if dloss is None:
            table = None
        else:
            dloss = dloss.float().contiguous()
        dlogits = _backward(rows, (*ctx.options, None, padding_mask, sequences), routes, dgates, table, dloss)
        return (dlogits, *[None] * 7)


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, counts, score, padding_mask, sequences):
        rows = _rows(logits)
        loss, table = _balance(rows, counts, score, padding_mask, sequences)
        ctx.score = score
        ctx.save_for_backward(rows, padding_mask, sequences, table)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        rows, padding_mask, sequences, table = ctx.saved_tensors
        dlogits = _backward(rows, (1, ctx.score, False, 1.0, None, padding_mask, sequences), None, None, table,
                            dloss.float().contiguous())
        return (dlogits, *[None] * 4)


def _balance(rows, counts, score, padding_mask, sequences):
    with torch.cuda.device(rows.device):
        router = _describe(rows, 1, score, False, 1.0, None, padding_mask, sequences)
        loss, table, workspace = _loss_buffers(router, rows.device)
        _lib.check(_lib.load().wm_balance_forward(
            ctypes.byref(router), _lib.ptr(counts), _lib.ptr(loss), _lib.ptr(table), _lib.ptr(workspace),
            workspace.numel(), _stream(rows, counts, padding_mask, sequences)))
    return loss, table


def _wants_gradient(logits):
    return torch.is_grad_enabled() and logits.requires_grad


def route_tokens(logits, top_k, *, score="softmax", renormalize=True, scale=1.0, bias=None, padding_mask=None):
    """Choose top_k experts for every token: (routes int32, gates float32), both [tokens, top_k].

    score        "softmax" over the token's experts, or "sigmoid" of each.
    renormalize  divide the chosen scores by their sum; `scale` multiplies the gates.
    bias         float32 [experts], added to the scores for the choice only (gates and gradients do not see it).
    padding_mask bool [tokens], True = padding: routes -1, gates 0, no gradient.
    A logit of -inf takes the expert out for that token; where fewer than top_k are left the rest are -1 with gate 0.
    Ties go to the lowest expert.  Gates are differentiable by the logits."""
    _check_logits(logits)
    _check_score(score)
    _check_choice(logits, top_k, scale)
    _check_vector(bias, "bias", (torch.float32,), logits.shape[1], logits)
    _check_vector(padding_mask, "padding_mask", (torch.bool, torch.uint8), logits.shape[0], logits)
    _require_device(logits, "logits")
    if not _wants_gradient(logits):
        return _route(_rows(logits), top_k, score, renormalize, scale, bias, padding_mask, None, False)[:2]
    return _Route.apply(logits, top_k, score, renormalize, scale, bias, padding_mask)


def expert_counts(routes, experts, *, sequences=None):
    """Routes per expert, int32 [experts], or [sequences, experts] with the sequences' offsets (int32
    [sequences + 1]).  Ids outside [0, experts) are "no route" and count nowhere."""
    if not isinstance(routes, torch.Tensor) or routes.ndim != 2 or routes.dtype != torch.int32:
        raise ValueError("routes must be an int32 tensor [tokens, top_k]")
    if not 1 <= routes.shape[1] <= MAX_TOP_K or not routes.is_contiguous():
        raise ValueError(f"routes must be contiguous, with 1 to {MAX_TOP_K} columns")
    if not isinstance(experts, int) or not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"experts must be in [1, {MAX_EXPERTS}]")
    _check_sequences(sequences, routes)
    _require_device(routes, "routes")
    with torch.cuda.device(routes.device):
        shape = (experts,) if sequences is None else (sequences.shape[0] - 1, experts)
        counts = torch.empty(shape, dtype=torch.int32, device=routes.device)
        _lib.check(_lib.load().wm_expert_counts(
            _lib.ptr(routes), routes.shape[0], routes.shape[1], experts, _lib.ptr(sequences),
            0 if sequences is None else sequences.shape[0] - 1, _lib.ptr(counts),
            _stream(routes, sequences)))
    return counts


def balance_loss(logits, counts, *, score="softmax", padding_mask=None, sequences=None):
    """The balance loss of a batch, a float32 scalar that is differentiable by the logits.

    With p the token's scores as shares of their sum, P_e the mean of p_e over the live tokens and
    f_e = experts * counts_e / sum(counts): sum over experts of f_e P_e; with `sequences` (int32 offsets,
    non-decreasing) the mean of that over the sequences that have a live token, counts then being [sequences, experts].
    counts come from `expert_counts`, possibly summed over ranks; they are taken as constants.  An even load gives 1."""
    _check_logits(logits)
    _check_score(score)
    _check_vector(padding_mask, "padding_mask", (torch.bool, torch.uint8), logits.shape[0], logits)
    _check_sequences(sequences, logits)
    shape = (logits.shape[1],) if sequences is None else (sequences.shape[0] - 1, logits.shape[1])
    if (not isinstance(counts, torch.Tensor) or counts.dtype != torch.int32 or tuple(counts.shape) != shape
            or counts.device != logits.device or not counts.is_contiguous()):
        raise ValueError(f"counts must be a contiguous int32 tensor {list(shape)} on the device of the logits")
    _require_device(logits, "logits")
    if not _wants_gradient(logits):
        return _balance(_rows(logits), counts, score, padding_mask, sequences)[0]
    return _Balance.apply(logits, counts, score, padding_mask, sequences)


def route_and_balance(logits, top_k, *, score="softmax", renormalize=True, scale=1.0, bias=None, padding_mask=None,
                      sequences=None):
    """`route_tokens`, `expert_counts` and `balance_loss` of those routes in one pass over the logits, and one for
    the gradient: (routes, gates, counts, loss).  Tokens that no sequence holds count as padding."""
    _check_logits(logits)
    _check_score(score)
    _check_choice(logits, top_k, scale)
    _check_vector(bias, "bias", (torch.float32,), logits.shape[1], logits)
    _check_vector(padding_mask, "padding_mask", (torch.bool, torch.uint8), logits.shape[0], logits)
    _check_sequences(sequences, logits)
    _require_device(logits, "logits")
    if not _wants_gradient(logits):
        return _route(_rows(logits), top_k, score, renormalize, scale, bias, padding_mask, sequences, True)[:4]
    return _RouteAndBalance.apply(logits, top_k, score, renormalize, scale, bias, padding_mask, sequences)
