"""CPU: argument checks of the FP8 matrix product's C entry (no CUDA call is reached) and of its Python layer."""
import ctypes

import pytest
import torch

from weftmoe_b200 import _lib
from weftmoe_b200.fp8 import fp8_linear, fp8_matmul, prepare_fp8_linear

GOOD = dict(aq=256, a_s=64, bq=256, bs=64, out=64, ld=16, m=8, n=16, k=128, a_rows=1, b_rows=128, f32=0, acc=0,
            room=None, room_bytes=0)


@pytest.mark.parametrize("change", [
    dict(m=-1), dict(n=-1), dict(k=-1), dict(a_rows=64), dict(b_rows=2), dict(ld=15), dict(acc=1),
    dict(aq=None), dict(a_s=None), dict(bq=None), dict(bs=None), dict(out=None), dict(aq=264), dict(bq=257),
    dict(a_s=66), dict(bs=65), dict(out=65), dict(out=66, f32=1),
])
def test_c_entry_refuses(change):
    lib = _lib.load()
    assert lib.wm_fp8_matmul(*{**GOOD, **change}.values(), None) == _lib.WM_ERR_INVALID
    assert "wm_fp8_matmul" in _lib.last_error()


@pytest.mark.parametrize("change", (dict(m=0), dict(n=0, ld=0), dict(m=0, out=None, aq=None)))
def test_nothing_to_do_touches_nothing(change):
    assert _lib.load().wm_fp8_matmul(*{**GOOD, **change}.values(), None) == _lib.WM_OK


def test_linear_entry_refuses():
    lib = _lib.load()
    for rows, k, n in ((-1, 128, 8), (4, -1, 8), (4, 128, -1)):
        assert lib.wm_fp8_linear(256, 0, rows, k, 256, 64, n, 64, 256, 1 << 20, None) == _lib.WM_ERR_INVALID
    assert lib.wm_fp8_linear(None, 0, 0, 128, None, None, 8, None, None, 0, None) == _lib.WM_OK
    size = ctypes.c_int64()
    assert lib.wm_fp8_matmul_workspace(-1, 1, 1, ctypes.byref(size)) == _lib.WM_ERR_INVALID
    assert lib.wm_fp8_linear_workspace(1, 1, -1, ctypes.byref(size)) == _lib.WM_ERR_INVALID


def test_status_entry_refuses_a_null_result():
    assert _lib.load().wm_fp8_matmul_status(ctypes.POINTER(ctypes.c_int32)(), None) == _lib.WM_ERR_INVALID


def test_python_layer_refuses_other_types():
    x = torch.zeros(4, 128)
    with pytest.raises(TypeError, match="FP8Tensor"):
        fp8_matmul(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        prepare_fp8_linear(x)
    with pytest.raises(TypeError, match="PreparedFP8Linear"):
        fp8_linear(x, x, x)
