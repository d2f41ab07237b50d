"""CPU: argument checks of the router operators (no CUDA call is reached), and the struct's layout."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from weftmoe_b200 import _lib
from weftmoe_b200.router import balance_loss, expert_counts, route_and_balance, route_tokens

ROOT = Path(__file__).resolve().parent.parent
LOGITS = torch.zeros(4, 8)


@pytest.mark.parametrize("call", (route_tokens, route_and_balance))
@pytest.mark.parametrize("change, words", [
    (dict(logits=torch.zeros(4, 8, dtype=torch.float64)), "BF16, FP32 or FP16"),
    (dict(logits=torch.zeros(2, 4, 8)), "BF16, FP32 or FP16"),
    (dict(logits=torch.zeros(4, 0)), "experts"),
    (dict(logits=torch.zeros(4, 1025)), "experts"),
    (dict(logits=torch.zeros(1, 1).expand(2 ** 26, 1)), "tokens"),
    (dict(top_k=0), "top_k"),
    (dict(top_k=9), "top_k"),
    (dict(logits=torch.zeros(4, 64), top_k=33), "top_k"),
    (dict(top_k=2.0), "top_k"),
    (dict(top_k=True), "top_k"),
    (dict(score="tanh"), "score"),
    (dict(scale=0.0), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(bias=torch.zeros(7)), "bias"),
    (dict(bias=torch.zeros(8, dtype=torch.bfloat16)), "bias"),
    (dict(padding_mask=torch.zeros(5, dtype=torch.bool)), "padding_mask"),
    (dict(padding_mask=torch.zeros(4)), "padding_mask"),
    (dict(padding_mask=torch.zeros(8, dtype=torch.bool)[::2]), "padding_mask"),
    ({}, "CUDA"),
])
def test_route_refusals(call, change, words):
    arguments = {"logits": LOGITS, "top_k": 2, **change}
    with pytest.raises(ValueError, match=words):
        call(arguments.pop("logits"), arguments.pop("top_k"), **arguments)


@pytest.mark.parametrize("sequences", (torch.zeros(3), torch.zeros(3, dtype=torch.int64),
                                       torch.zeros(1, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)))
def test_sequences_are_int32_offsets(sequences):
    with pytest.raises(ValueError, match="sequences"):
        route_and_balance(LOGITS, 2, sequences=sequences)
    with pytest.raises(ValueError, match="sequences"):
        expert_counts(torch.zeros(4, 2, dtype=torch.int32), 8, sequences=sequences)


def test_counts_refusals():
    routes = torch.zeros(4, 2, dtype=torch.int32)
    for bad in (routes.long(), routes[0], routes.t(), torch.zeros(4, 33, dtype=torch.int32)):
        with pytest.raises(ValueError, match="routes"):
            expert_counts(bad, 8)
    with pytest.raises(ValueError, match="tokens"):
        expert_counts(torch.empty((2 ** 26, 1), dtype=torch.int32, device="meta"), 8)
    for experts in (0, 1025, 8.0):
        with pytest.raises(ValueError, match="experts"):
            expert_counts(routes, experts)
    with pytest.raises(ValueError, match="CUDA"):
        expert_counts(routes, 8)


def test_balance_refusals():
    counts = torch.zeros(8, dtype=torch.int32)
    offsets = torch.tensor([0, 2, 4], dtype=torch.int32)
    for bad in (counts[:7], counts.long(), counts[None], torch.zeros(16, dtype=torch.int32)[::2], None):
        with pytest.raises(ValueError, match="counts"):
            balance_loss(LOGITS, bad)
    with pytest.raises(ValueError, match="counts"):
        balance_loss(LOGITS, counts, sequences=offsets)
    with pytest.raises(ValueError, match="score"):
        balance_loss(LOGITS, counts, score="relu")
    with pytest.raises(ValueError, match="CUDA"):
        balance_loss(LOGITS, counts)


def _description(**change):
    fields = dict(logits=64, row_stride=8, dtype=1, tokens=4, experts=8, top_k=2, score=0, renormalize=1, scale=1.0,
                  num_sequences=0, bias=None, padding=None, sequences=None)
    return _lib.WmRouter(**{**fields, **change})


def test_c_entries_refuse_before_any_device_work():
    lib = _lib.load()
    size = ctypes.c_int64()
    for change in (dict(experts=0), dict(experts=1025, row_stride=1025), dict(dtype=3), dict(row_stride=7),
                   dict(score=2), dict(tokens=-1), dict(tokens=2 ** 26), dict(logits=None), dict(num_sequences=2),
                   dict(sequences=64, num_sequences=0), dict(sequences=64, num_sequences=65536)):
        r = _description(**change)
        assert lib.wm_router_workspace(ctypes.byref(r), ctypes.byref(size)) == _lib.WM_ERR_INVALID, change
        assert lib.wm_router_forward(ctypes.byref(r), 64, 64, None, None, None, None, 0, None) == _lib.WM_ERR_INVALID
    good = _description()
    assert lib.wm_router_workspace(ctypes.byref(good), ctypes.byref(size)) == _lib.WM_OK and size.value > 0
    # outputs and workspaces that are missing, small or misaligned
    assert lib.wm_router_forward(ctypes.byref(good), None, 64, None, None, None, None, 0, None) == _lib.WM_ERR_INVALID
    for workspace, held in ((64, size.value - 1), (72, size.value), (None, size.value)):
        assert lib.wm_router_forward(ctypes.byref(good), 64, 64, 64, 64, 64, workspace, held,
                                     None) == _lib.WM_ERR_INVALID
        assert lib.wm_balance_forward(ctypes.byref(good), 64, 64, 64, workspace, held, None) == _lib.WM_ERR_INVALID
    for change in (dict(top_k=0), dict(top_k=9), dict(scale=0.0), dict(scale=float("nan"))):
        r = _description(**change)
        assert lib.wm_router_forward(ctypes.byref(r), 64, 64, None, None, None, None, 0, None) == _lib.WM_ERR_INVALID
        assert lib.wm_router_backward(ctypes.byref(r), 64, 64, None, None, 64, None) == _lib.WM_ERR_INVALID
    for pair in ((64, None, None, None), (None, None, 64, None), (None, None, None, None)):
        assert lib.wm_router_backward(ctypes.byref(good), *pair, 64, None) == _lib.WM_ERR_INVALID
    # addresses that are not multiples of their elements (the table's: of 16 bytes)
    for change in (dict(logits=66), dict(logits=65, dtype=0), dict(logits=65, dtype=2), dict(bias=66),
                   dict(sequences=66, num_sequences=1)):
        r = _description(**change)
        assert lib.wm_router_workspace(ctypes.byref(r), ctypes.byref(size)) == _lib.WM_ERR_INVALID, change
        assert lib.wm_router_backward(ctypes.byref(r), 64, 64, None, None, 64, None) == _lib.WM_ERR_INVALID, change
    for outputs in ((66, 64, None, None, None, None, 0), (64, 65, None, None, None, None, 0),
                    (64, 64, 66, 64, 64, 64, size.value), (64, 64, 64, 65, 64, 64, size.value),
                    (64, 64, 64, 64, 66, 64, size.value)):
        assert lib.wm_router_forward(ctypes.byref(good), *outputs, None) == _lib.WM_ERR_INVALID, outputs
    for given in ((66, 64, 64), (64, 66, 64), (64, 64, 66)):
        assert lib.wm_balance_forward(ctypes.byref(good), *given, 64, size.value, None) == _lib.WM_ERR_INVALID, given
    for pairs in ((66, 64, None, None, 64), (64, 66, None, None, 64), (None, None, 68, 64, 64), (None, None, 64, 66, 64),
                  (64, 64, None, None, 66)):
        assert lib.wm_router_backward(ctypes.byref(good), *pairs, None) == _lib.WM_ERR_INVALID, pairs
    for routes, sequences, counts in ((66, None, 64), (64, 66, 64), (64, None, 65)):
        assert lib.wm_expert_counts(routes, 4, 2, 8, sequences, int(sequences is not None), counts,
                                    None) == _lib.WM_ERR_INVALID
    assert lib.wm_expert_counts(64, 4, 33, 8, None, 0, 64, None) == _lib.WM_ERR_INVALID
    assert lib.wm_expert_counts(None, 4, 2, 8, None, 0, 64, None) == _lib.WM_ERR_INVALID


def test_struct_matches_the_header(tmp_path):
    header = ROOT / "include" / "weftmoe_b200.h"
    lines = ["#include <stdio.h>", f'#include "{header}"', "int main(void) {",
             '  printf("size %zu\\n", sizeof(wm_router));']
    lines += [f'  printf("{name} %zu\\n", offsetof(wm_router, {name}));' for name, _ in _lib.WmRouter._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    text = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    found = dict(line.split() for line in text.splitlines())
    assert int(found.pop("size")) == ctypes.sizeof(_lib.WmRouter)
    assert {k: int(v) for k, v in found.items()} == {n: getattr(_lib.WmRouter, n).offset for n, _ in
                                                     _lib.WmRouter._fields_}
