"""GPU: large FP8 products on CTA pairs, and where those cannot be taken.  Whole-number operands: sums are exact."""
import ctypes

import pytest
import torch

from tests.test_gpu_fp8_matmul import operand, wide
from weftmoe_b200 import _lib
from weftmoe_b200.fp8 import fp8_linear, fp8_matmul, poll_fp8_matmul, prepare_fp8_linear

pytestmark = pytest.mark.gpu

M, N, K = 1500, 1700, 2000


def workspace(m, n, k):
    size = ctypes.c_int64()
    assert _lib.load().wm_fp8_matmul_workspace(m, n, k, ctypes.byref(size)) == _lib.WM_OK
    return size.value


@pytest.fixture
def too_few_registers():
    lib = _lib.load()
    assert workspace(M, N, K) > 0                                 # as built, these sizes go to pairs
    lib.wm_debug_matmul_pair_registers(167)
    yield
    lib.wm_debug_matmul_pair_registers(0)


@pytest.mark.parametrize("a_rows, b_rows", [(1, 1), (1, 128), (128, 128)])
def test_products_without_pairs(a_rows, b_rows, too_few_registers):
    """Pair kernels built with too few registers are not launched, with or without a workspace: the one-CTA kernels
    take the product."""
    assert workspace(M, N, K) == 0
    a, b = operand(M, K, a_rows, 60), operand(N, K, b_rows, 61)
    want = (wide(a) @ wide(b).t()).float()
    assert torch.equal(fp8_matmul(a, b, dtype=torch.float32), want)
    out, room = torch.empty(M, N, device="cuda"), torch.empty(1 << 20, device="cuda", dtype=torch.uint8)
    code = _lib.load().wm_fp8_matmul(a.data.data_ptr(), a.scales.data_ptr(), b.data.data_ptr(), b.scales.data_ptr(),
                                     out.data_ptr(), N, M, N, K, a_rows, b_rows, 1, 0, room.data_ptr(), room.numel(),
                                     torch.cuda.current_stream().cuda_stream)
    assert code == _lib.WM_OK and torch.equal(out, want)
    poll_fp8_matmul()


def test_projection_without_pairs(too_few_registers):
    weight = torch.randint(-4, 5, (N, K), device="cuda").bfloat16()
    x = torch.randint(-4, 5, (M, K), device="cuda").bfloat16()
    y = fp8_linear(x, weight, prepare_fp8_linear(weight, training=False))
    assert torch.equal(y, (x.double() @ weight.double().t()).bfloat16())


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("a_rows, b_rows", [(128, 1), (128, 128)])
@pytest.mark.parametrize("m, n, k", [(M, N, K), (1408, 1665, 2048), (4100, 4200, 640)])
def test_packed_scales_of_128_rows_on_the_left(m, n, k, a_rows, b_rows, dtype):
    """Power-of-two scales of 128 rows of A on the tensor cores, also where the last 128 or 256 rows are not full."""
    assert workspace(m, n, k) > 0
    a, b = operand(m, k, a_rows, 62), operand(n, k, b_rows, 63)
    assert torch.equal(fp8_matmul(a, b, dtype=dtype), (wide(a) @ wide(b).t()).float().to(dtype))
    poll_fp8_matmul()


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("m, n, pitch", [(130, 517, 520), (130, 65, 72), (300, 1001, 1008), (1500, 1701, 1704), (4100, 4199, 4200)])
def test_results_of_odd_width_in_aligned_rows(m, n, pitch, dtype):
    """Rows that start on 16 bytes and end between: what lies behind them stays."""
    a, b = operand(m, 640, 1, 64), operand(n, 640, 128, 65)
    holder = torch.full((m, pitch), 7.0, dtype=dtype, device="cuda")
    fp8_matmul(a, b, dtype=dtype, out=holder[:, :n])
    assert torch.equal(holder[:, :n], (wide(a) @ wide(b).t()).float().to(dtype))
    assert (holder[:, n:] == 7).all()
