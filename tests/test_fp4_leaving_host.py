"""When a block of the 4-bit products may leave, read from the source (no GPU needed: a wait that runs out in them
takes a fault to bring about)."""

import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "x-minimaxh3_b200", "csrc", "fp4_gemm.cu")


def _kernel(name):
    code = re.sub(r"//[^\n]*", "", open(SOURCE).read())
    start = code.index(name + "(const")
    return re.sub(r"\s+", " ", code[start: code.index("template <int FORMAT", start)])


def test_a_block_that_gave_up_stays_for_the_others_sums():
    """Others may still write their sums into its shared memory: it waits for them at the cluster's barrier, which counts
    blocks that have left.  Those that have everything do not wait."""
    body = _kernel("fp4_split_kernel")
    end = body[body.rindex("__syncthreads();"):]
    assert "if (split > 1 && abort_flag) { cluster_arrive(); cluster_wait(); }" in end
    assert "mbar_wait_sent(&sent, &abort_flag)" in body  # which raises the flag
