"""CPU: a kernel's tcgen05 instructions name one CTA group.  PTX asks for the same `.cta_group` in all of a kernel's
tcgen05 instructions that carry the qualifier, the allocation of TMEM among them."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "weftmoe_b200" / "csrc"
TMEM_CALL = re.compile(r"\btmem_(alloc|relinquish|dealloc)(<[^>]*>)?\(")


def text_of(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def tmem_calls(name):
    return [(m.group(1), m.group(2)) for m in TMEM_CALL.finditer(text_of(name))]


def test_tmem_helpers_come_in_both_groups():
    text = text_of("ptx.cuh")
    for instruction in ("alloc", "relinquish_alloc_permit", "dealloc"):
        for group in (1, 2):
            assert f"tcgen05.{instruction}.cta_group::{group}.sync.aligned" in text, (instruction, group)


@pytest.mark.parametrize("name, group", [("fp8_matmul.cu", "<PAIR ? 2 : 1>"), ("gemm2.cuh", "<2>")])
def test_pair_kernels_take_their_tmem_as_a_pair(name, group):
    calls = tmem_calls(name)
    assert sorted(c for c, _ in calls) == ["alloc", "dealloc", "relinquish"]
    assert all(given == group for _, given in calls), calls


def test_one_cta_kernels_name_one_cta():
    """Files without an instruction for a pair take the helpers as they are by default."""
    for path in sorted(CSRC.glob("*.cu*")):
        if path.name != "ptx.cuh" and "_pair(" not in text_of(path.name):
            assert all(given is None for _, given in tmem_calls(path.name)), path.name
