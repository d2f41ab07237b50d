"""GPU: storage that a call of another stream still uses is not handed out again."""
import pytest
import torch

from weftmoe_b200.fp8 import FP8Tensor, fp8_matmul

pytestmark = pytest.mark.gpu


def ones(rows, k, block_rows):
    return FP8Tensor(torch.ones(rows, k, device="cuda").to(torch.float8_e4m3fn),
                     torch.ones(-(-rows // block_rows), k // 128, device="cuda"), (rows, k), block_rows)


@pytest.mark.parametrize("accumulate", (False, True))
@pytest.mark.parametrize("m", (8, 1500))
def test_a_given_out_stays_until_the_product_has_used_it(m, accumulate):
    """`out` comes from another stream's part of the allocator and is released while the product waits for its turn:
    that stream must not get the memory again before the product is done."""
    a, b = ones(m, 256, 1), ones(1700, 256, 128)
    fp8_matmul(a, b)
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        out = torch.zeros(m, 1700, device="cuda")
        reference = out.clone()
    torch.cuda.synchronize()
    address = out.data_ptr()
    torch.cuda._sleep(100_000_000)                        # about 50 ms before the product's turn
    fp8_matmul(a, b, dtype=torch.float32, out=out, accumulate=accumulate)
    busy = torch.cuda.Event()
    busy.record()
    del out
    with torch.cuda.stream(other):
        again = torch.empty_like(reference)
    assert not busy.query(), "the stream was done before the check"
    assert again.data_ptr() != address
    torch.cuda.synchronize()
