"""The debug-checked build (-DWB200_CHECKS) covers the kernels beside frozen weights: each tests an index in front of its stores, and none of the tests below
fails a predicate when they run against it."""

import os
import re
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "wave_b200" / "csrc"

# a store that goes through one of these is tested in it
HELPERS = ("tma_store_2d", "finish_hidden", "sum_slices")


@pytest.mark.parametrize("source", ["adapters.cuh", "router.cuh", "input_grad_sm100.cuh"])
def test_every_kernel_tests_its_stores(source):
    """Read from the sources, without a GPU. (The router's second launch writes one number an expert and two scalars.)"""
    text = re.sub(r"//[^\n]*", "", (CSRC / source).read_text())
    parts = text.split("__global__")[1:]
    assert parts
    for part in parts:
        name = re.search(r"(\w+_kernel)\s*\(", part).group(1)
        assert "WB_CHECK(" in part or any(h in part for h in HELPERS), f"{name} stores without a check"


@pytest.mark.gpu
def test_no_predicate_fails_under_the_debug_checked_build():
    lib = ROOT / "wave_b200" / "libwave_b200_checks.so"
    if not lib.exists():
        pytest.fail("libwave_b200_checks.so is missing: run `python -m wave_b200.build --checks` (build() makes it)")
    cases = ["test_gpu_adapters_exact.py", "test_gpu_input_grad.py", "test_gpu_router.py"]
    res = subprocess.run([sys.executable, "-m", "pytest", "-q", "-m", "gpu", "-p", "no:cacheprovider", *(str(ROOT / "tests" / c) for c in cases)], cwd=ROOT,
                         env=dict(os.environ, WAVE_B200_LIB=str(lib)), capture_output=True, text=True, timeout=600)
    assert res.returncode == 0 and "no predicate failed" in res.stdout, res.stdout[-3000:] + res.stderr[-2000:]
