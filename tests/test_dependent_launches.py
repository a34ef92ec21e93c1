"""The order in which the kernels beside frozen weights wait for the kernel before them and release the one behind them, read from their sources: runs
without a GPU.

What a kernel reads before its own wait has to be older than the kernel before it. That holds for a call's first kernel only if nothing released it
early, and for the kernel behind a call only if the call's first kernel waited before it let others begin."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "wave_b200" / "csrc"

# launched behind another kernel of the same call, which has waited
FOLLOWERS = {"adapter_expand_few_kernel", "adapter_expand_few_whole_kernel", "adapter_expand_tile_kernel", "router_finish_kernel"}


def kernels(name):
    """(name, body) of every kernel of a source, without comments."""
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    for part in text.split("__global__")[1:]:
        yield re.search(r"(\w+_kernel)\s*\(", part).group(1), part


@pytest.mark.parametrize("source", ["adapters.cuh", "router.cuh", "input_grad_sm100.cuh"])
def test_the_first_kernel_of_a_call_waits_before_it_releases(source):
    seen = set()
    for name, body in kernels(source):
        seen.add(name)
        wait, release = body.find("pdl_wait("), body.find("pdl_launch_dependents(")
        assert wait >= 0 and release >= 0, name
        assert name in FOLLOWERS or wait < release, f"{name} releases its dependents before it has waited"
    assert len(seen) >= 1 and (source != "adapters.cuh" or "adapter_outer_kernel" in seen)


def test_followers_are_launched_behind_another_kernel():
    """The expansions are launched by run_expand, which both entries call behind run_shrink; the router's second launch is in its entry."""
    text = re.sub(r"//[^\n]*", "", (CSRC / "adapt.cu").read_text())
    calls = [m.start() for m in re.finditer(r"run_expand\(c,", text)]
    shrinks = [m.start() for m in re.finditer(r"run_shrink\(c,", text)]
    assert len(calls) == len(shrinks) == 2 and all(s < c for s, c in zip(shrinks, calls))
    assert text.index("launch(kernel, dim3(ctas)") < text.index("wb::router_finish_kernel")
