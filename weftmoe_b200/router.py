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
import functools
import math

import torch

from . import _lib
from ._launch import on_device, stream_of

_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
_SCORES = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS = 1024
MAX_TOP_K = 32
MAX_TOKENS = 2 ** 26 - 1
MAX_SEQUENCES = 65535


def _check_logits(logits):
    if not isinstance(logits, torch.Tensor) or logits.ndim != 2 or logits.dtype not in _DTYPES:
        raise ValueError("logits must be a BF16, FP32 or FP16 tensor [tokens, experts]")
    if not 1 <= logits.shape[1] <= MAX_EXPERTS:
        raise ValueError(f"logits must have 1 to {MAX_EXPERTS} experts")
    if logits.shape[0] > MAX_TOKENS:
        raise ValueError(f"logits must have at most {MAX_TOKENS} tokens")


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


@functools.lru_cache(maxsize=256)
def _workspace_bytes(tokens, experts, num_sequences):
    router = _lib.WmRouter(logits=16, row_stride=experts, dtype=1, tokens=tokens, experts=experts,
                           num_sequences=num_sequences, sequences=16 if num_sequences else None)
    size = ctypes.c_int64()
    _lib.check(_lib.load().wm_router_workspace(ctypes.byref(router), ctypes.byref(size)))
    return size.value


def _loss_buffers(logits, router):
    """(loss, table, workspace) of a call that computes the loss."""
    sequences = router.num_sequences
    return (logits.new_empty((), dtype=torch.float32),
            logits.new_empty(max(1, sequences) * router.experts + 1, dtype=torch.float32),
            logits.new_empty(_workspace_bytes(router.tokens, router.experts, sequences), dtype=torch.uint8))


def _address(tensor):
    return None if tensor is None else tensor.data_ptr()


def _plain_gradient(gradient):
    """An incoming gradient as contiguous FP32 (broadcast ones are expanded)."""
    if gradient is None or (gradient.dtype == torch.float32 and gradient.is_contiguous()):
        return gradient
    return gradient.float().contiguous()


def _backward(logits, router_args, routes, dgates, table, dloss):
    if torch.is_grad_enabled():
        raise RuntimeError("The router's gradients cannot be differentiated again")
    dgates, dloss = _plain_gradient(dgates), _plain_gradient(dloss)
    device = logits.device
    with on_device(device):
        dlogits = logits.new_empty(logits.shape)
        router = _describe(logits, *router_args)
        _lib.check(_lib.load().wm_router_backward(
            ctypes.byref(router), _address(routes), _address(dgates), _address(table), _address(dloss),
            dlogits.data_ptr(), stream_of(device, logits, *router_args[-2:], routes, dgates, table, dloss)))
    return dlogits


def _route(logits, top_k, score, renormalize, scale, bias, padding_mask, sequences, balance):
    """(routes, gates, counts, loss, table); the last three are None without the loss."""
    device = logits.device
    tokens, experts = logits.shape
    with on_device(device):
        routes = logits.new_empty((tokens, top_k), dtype=torch.int32)
        gates = logits.new_empty((tokens, top_k), dtype=torch.float32)
        router = _describe(logits, top_k, score, renormalize, scale, bias, padding_mask, sequences)
        counts = loss = table = workspace = None
        if balance:
            loss, table, workspace = _loss_buffers(logits, router)
            counts = logits.new_empty((experts,) if sequences is None else (router.num_sequences, experts),
                                      dtype=torch.int32)
        _lib.check(_lib.load().wm_router_forward(
            ctypes.byref(router), routes.data_ptr(), gates.data_ptr(), _address(counts), _address(loss),
            _address(table), _address(workspace), 0 if workspace is None else workspace.numel(),
            stream_of(device, logits, bias, padding_mask, sequences)))
    return routes, gates, counts, loss, table


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, score, renormalize, scale, bias, padding_mask):
        rows = _rows(logits)
        routes, gates, *_ = _route(rows, top_k, score, renormalize, scale, bias, padding_mask, None, False)
        ctx.options = (top_k, score, renormalize, scale)
        ctx.save_for_backward(rows, routes, padding_mask)
        ctx.mark_non_differentiable(routes)
        ctx.set_materialize_grads(False)   # no zeros for the routes
        return routes, gates

    @staticmethod
    def backward(ctx, _, dgates):
        if dgates is None:
            return (None,) * 7
        rows, routes, padding_mask = ctx.saved_tensors
        dlogits = _backward(rows, (*ctx.options, None, padding_mask, None), routes,
                            dgates, None, None)
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
    def backward(ctx, _routes, dgates, _counts, dloss):
        rows, routes, padding_mask, sequences, table = ctx.saved_tensors
        if dgates is None and dloss is None:
            return (None,) * 8
        if dgates is None:
            routes = None
        if dloss is None:
            table = None
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
    def backward(ctx, dloss):
        rows, padding_mask, sequences, table = ctx.saved_tensors
        dlogits = _backward(rows, (1, ctx.score, False, 1.0, None, padding_mask, sequences), None, None, table,
                            dloss)
        return (dlogits, *[None] * 4)


def _balance(rows, counts, score, padding_mask, sequences):
    device = rows.device
    with on_device(device):
        router = _describe(rows, 1, score, False, 1.0, None, padding_mask, sequences)
        loss, table, workspace = _loss_buffers(rows, router)
        _lib.check(_lib.load().wm_balance_forward(
            ctypes.byref(router), counts.data_ptr(), loss.data_ptr(), table.data_ptr(), workspace.data_ptr(),
            workspace.numel(), stream_of(device, rows, counts, padding_mask, sequences)))
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
    if routes.shape[0] > MAX_TOKENS:
        raise ValueError(f"routes must have at most {MAX_TOKENS} tokens")
    if not isinstance(experts, int) or not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"experts must be in [1, {MAX_EXPERTS}]")
    _check_sequences(sequences, routes)
    _require_device(routes, "routes")
    device = routes.device
    with on_device(device):
        counts = routes.new_empty((experts,) if sequences is None else (sequences.shape[0] - 1, experts))
        _lib.check(_lib.load().wm_expert_counts(
            routes.data_ptr(), routes.shape[0], routes.shape[1], experts, _address(sequences),
            0 if sequences is None else sequences.shape[0] - 1, counts.data_ptr(),
            stream_of(device, routes, sequences)))
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
