"""CPU: sizes that the C ABI's 32 bits do not hold are refused; they used to arrive cut to 32 bits, as a smaller problem."""
import pytest
import torch

from weftmoe_b200 import _lib, fp8
from weftmoe_b200.fp8 import prepare_fp8_linear

FAR = 2 ** 32 + 8
WORDS = r"2\^31"


@pytest.mark.parametrize("shape", [(1, FAR), (FAR, 1), (1, 2 ** 31), (2, 3, FAR), (FAR, 2, 3)])
def test_sources_of_the_quantisers(shape):
    with pytest.raises(ValueError, match=WORDS):
        fp8._source_args(torch.empty(shape, dtype=torch.bfloat16, device="meta"))


def test_the_largest_size_passes():
    assert fp8._source_args(torch.empty(2 ** 31 - 1, 1, dtype=torch.float32, device="meta"))[1:] == (1, 1, 2 ** 31 - 1, 1)


@pytest.mark.parametrize("sizes", [(FAR, 8, 128), (8, FAR, 128), (8, 8, FAR)])
def test_products(sizes):
    empty = torch.empty(0)
    with pytest.raises(ValueError, match=WORDS):
        _lib.binding().fp8_matmul(empty, empty, 1, empty, empty, 128, *sizes, False, None, False)


@pytest.mark.parametrize("x, weight", [((FAR, 1), (8, 1)), ((8, FAR), (8, FAR)), ((8, 1), (FAR, 1))])
def test_projections(x, weight):
    empty = torch.empty(0)
    x, weight = (torch.zeros(1, 1).expand(shape) for shape in (x, weight))
    with pytest.raises(ValueError, match=WORDS):
        _lib.binding().fp8_linear(x, weight, empty, empty, None, None)


def test_imported_weights():
    with pytest.raises(ValueError, match=WORDS):
        prepare_fp8_linear(fp8._allocate((1, FAR), 128, torch.empty(0, device="meta")))
