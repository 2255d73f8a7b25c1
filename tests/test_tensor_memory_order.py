"""Who takes tensor memory and lets the next launch start early: the order of the two in every kernel, read from the sources (no GPU).

A launch that starts early may ask for tensor memory ahead of its wait for the launch in front.  If a block of that launch has yet to ask for its own, the two
wait for each other, and neither wait is bounded.
"""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "project_maya_b200" / "csrc"


def kernels():
    for path in sorted(CSRC.glob("*.cu*")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for body in text.split("__global__")[1:]:
            if "tmem_alloc(" in body:
                yield pytest.param(body, id=path.name + ":" + re.search(r"(\w+)\s*\(\s*(?:const|$)", re.sub(r"__\w+__(?:\([^)]*\))?", "", body)).group(1))


def test_there_are_such_kernels():
    assert len(list(kernels())) >= 4


@pytest.mark.parametrize("body", list(kernels()))
def test_tensor_memory_comes_before_the_signal(body):
    """In the text: asked for above every signal, and between the two a barrier of the block, or the signal is that of the warp that asked."""
    ask, signal = body.index("tmem_alloc("), body.find("grid_launch_dependents(")
    assert signal < 0 or ask < signal
    own = re.search(r"if \(warp == \w+\) \{\s*tmem_alloc\([^;]*\);\s*grid_launch_dependents\(\);\s*\}", body)
    assert signal < 0 or own or "__syncthreads()" in body[ask:signal]
