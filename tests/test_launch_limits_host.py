"""What a launch changes of a kernel for everyone (no GPU needed)."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "x-minimaxh3_b200", "csrc")


def test_limits_of_shared_memory_are_constants():
    """A kernel's limit holds for all host threads: one that was set to a call's own size could be lowered by another
    thread before that call's launch."""
    found = 0
    for name in sorted(os.listdir(CSRC)):
        code = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
        for size in re.findall(r"cudaFuncAttributeMaxDynamicSharedMemorySize,\s*([^;]*?)\);", code):
            assert re.fullmatch(r"(\w+(<\w+>)?::)?k[A-Z]\w*", size), (name, size)
            found += 1
    assert found
