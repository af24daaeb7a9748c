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


def test_a_pair_waits_for_the_copies_of_both():
    """The even block's barriers count both blocks' copies, but only up to its own last fill.  The odd one waits for its
    own last fills to be used, which its own barriers are told: the even one may have given up before them."""
    body = _kernel("fp4_pair_kernel")
    producer = body[body.index("if (warp == 0) {"): body.index("} else if (warp == 1) {")]
    last = producer[producer.rindex("for ("):]
    assert "uint64_t* landed = rank == 0 ? full : empty;" in producer
    assert "mbar_wait_warp(&landed[s], s < fill.stage ? fill.parity : fill.parity ^ 1u, &late_flag" in last


def test_the_parity_of_a_stages_last_fill():
    """Of a ring of stages filled `fills` times in all, the parity that the wait above computes is that of the last
    phase of each stage, or, of a stage never filled, one that a new barrier takes as over."""
    for stages in (1, 2, 5):
        for fills in range(4 * stages):
            stage = parity = 0
            count = [0] * stages
            for _ in range(fills):
                count[stage] += 1
                stage += 1
                if stage == stages:
                    stage, parity = 0, parity ^ 1
            for s in range(stages):
                waits = parity if s < stage else parity ^ 1
                assert waits == (count[s] - 1) % 2  # phases are counted from 0; -1 is the one before the first
