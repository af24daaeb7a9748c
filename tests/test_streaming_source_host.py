"""Rules of the streaming kernels that no run can show (no GPU needed)."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "x-minimaxh3_b200", "csrc")
CHAINED = ("window_attn.cu", "decode_attn.cu", "kv_pages.cu", "streaming.cuh")


def _code(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def test_chained_kernels_use_no_read_only_loads():
    """A kernel that starts while the one before it runs may not load what that one writes through the
    read-only path, which asks for memory that stays as it is for the kernel's whole time."""
    for name in CHAINED:
        assert not re.search(r"ld\.global(\.\w+)*\.nc|__ldg\b|__restrict__", _code(name)), name


def test_chained_kernels_wait_before_they_touch_memory():
    """Each kernel of these files lets the next one start and then waits for the one before it."""
    for name in CHAINED[:3]:
        code = _code(name)
        kernels = len(re.findall(r"__global__", code))
        assert kernels == len(re.findall(r"chain_next\(\);\s*chain_wait\(\);", code)) > 0, name
