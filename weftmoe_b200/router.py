"""Router operators in front of `TensorRuntime` / `moe`: top-k routes with gates, per-expert counts, balance loss.

    routes, gates = route_tokens(logits, top_k)                        # what forward / moe take
    counts = expert_counts(routes, experts)                            # int32 load of each expert
    loss = balance_loss(logits, counts)                                # routes of this or of another router
    routes, gates, counts, loss = route_and_balance(logits, top_k)     # all of it in one pass over the logits

The reference leaves the router to its host framework (weftmoe/megatron.py:164-188 takes routes and gates from it);
the definitions are in include/weftmoe_b200.h beside `wm_router`.  All arithmetic runs in libweftmoe_b200.so; this
file checks arguments, binding/torch_binding.cpp allocates results and joins the calls to autograd.  Every call enqueues on the current
stream of the logits' device, synchronises nothing and may be captured in a CUDA graph; capture a backward pass
together with its forward pass (autograd runs a backward pass on the stream of its forward pass).  First derivatives in
reverse mode: forward mode and second derivatives are refused.
"""
from __future__ import annotations

import math

import torch

from . import _lib

_DTYPES = (torch.bfloat16, torch.float32, torch.float16)
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


def route_tokens(logits, top_k, *, score="softmax", renormalize=True, scale=1.0, bias=None, padding_mask=None):
    """Choose top_k experts for every token: (routes int32, gates float32), both [tokens, top_k].

    score        "softmax" over the token's experts, or "sigmoid" of each.
    renormalize  divide the chosen scores by their sum; `scale` multiplies the gates.
    bias         finite float32 [experts], added to the scores for the choice only (gates and gradients do not see it).
    padding_mask bool [tokens], True = padding: routes -1, gates 0, no gradient.
    A logit of -inf takes the expert out for that token; where fewer than top_k are left the rest are -1 with gate 0.
    Ties go to the lowest expert.  Gates are differentiable by the logits."""
    _check_logits(logits)
    _check_score(score)
    _check_choice(logits, top_k, scale)
    _check_vector(bias, "bias", (torch.float32,), logits.shape[1], logits)
    _check_vector(padding_mask, "padding_mask", (torch.bool, torch.uint8), logits.shape[0], logits)
    _require_device(logits, "logits")
    return tuple(_lib.binding().route(logits, top_k, _SCORES[score], renormalize, scale, bias, padding_mask, None, False))


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
    return _lib.binding().expert_counts(routes, experts, sequences)


def balance_loss(logits, counts, *, score="softmax", padding_mask=None, sequences=None):
    """The balance loss of a batch, a float32 scalar that is differentiable by the logits.

    With p the token's scores as shares of their sum, P_e the mean of p_e over the live tokens and
    f_e = experts * counts_e / sum(counts): sum over experts of f_e P_e (tokens without an available expert are left out);
    with `sequences` (int32 offsets, non-decreasing) the mean of that over the sequences that have a live token, counts then being [sequences, experts].
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
    return _lib.binding().balance(logits, counts, _SCORES[score], padding_mask, sequences)


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
    return tuple(_lib.binding().route(logits, top_k, _SCORES[score], renormalize, scale, bias, padding_mask, sequences,
                                      True))
