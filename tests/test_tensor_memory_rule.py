"""Kernels that allocate tensor memory keep each other off an SM by the shared memory they ask for, and say so to the compiler: read from the sources, runs
without a GPU. (A kernel that holds columns while it waits for its cluster, next to one of another stream that does the same, could wait for good.)"""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "wave_b200" / "csrc"
SOURCES = {p.name: re.sub(r"//[^\n]*", "", p.read_text()) for p in sorted(CSRC.glob("*.cuh"))}
ALLOCATING = [name for name, text in SOURCES.items() if name != "ptx.cuh" and "tmem_alloc<" in text]


def test_the_kernels_are_found():
    assert {"gemm_sm100.cuh", "input_grad_sm100.cuh", "adapters.cuh", "skinny_sm100.cuh"} <= set(ALLOCATING)
    assert "kSmemOfTmemKernel = 160 * 1024" in SOURCES["ptx.cuh"] and not any("tmem_alloc<" in (CSRC / n).read_text() for n in ("api.cu", "adapt.cu"))


@pytest.mark.parametrize("name", ALLOCATING)
def test_each_states_its_shared_memory(name):
    text = SOURCES[name]
    stated = re.findall(r"static_assert\([^;]*SMEM_BYTES[^;]*kSmemOfTmemKernel", text)
    assert len(stated) >= len(re.findall(r"tmem_alloc<", text)), name
