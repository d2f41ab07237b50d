"""CPU: a kernel that starts under the one before it (programmatic launch) reads what that one writes by ordinary loads.
Loads through the read-only path (__ldg, or const __restrict__ parameters of a kernel) are for memory that nothing writes
while the kernel runs, from its start and not from its wait on."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "weftmoe_b200" / "csrc"


def kernel(name, path):
    """(parameters, body) of the kernel's definition."""
    text = re.sub(r"//[^\n]*", "", (CSRC / path).read_text())
    start = re.search(rf"\n{name}\(", text).end()
    brace = text.index("{", start)
    depth, end = 0, brace
    for end in range(brace, len(text)):
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        if depth == 0:
            break
    return text[start:brace], text[brace:end]


@pytest.mark.parametrize("name, path", [("pack_scales_kernel", "fp8_matmul.cu"), ("fp8_matmul_kernel", "fp8_matmul.cu")])
def test_waits_and_then_loads_in_the_ordinary_way(name, path):
    parameters, body = kernel(name, path)
    assert "cudaGridDependencySynchronize();" in body
    before, after = body.split("cudaGridDependencySynchronize();")
    assert "__restrict__" not in parameters and "__ldg(" not in body
    assert not re.search(r"\bscales\s*\[|p_scales\s*\[|tma_load", before)


def test_the_summing_kernel_reads_its_records_in_the_ordinary_way():
    """Its sequences and given counts are complete before the kernel in front of it starts."""
    _, body = kernel("balance_finish_kernel", "router.cu")
    before, after = body.split("cudaGridDependencySynchronize();")
    assert "rec." not in before and not re.search(r"__ldg\((?!a\.sequences)", after)
