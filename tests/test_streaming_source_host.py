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


def test_window_kernel_waits_for_what_it_started():
    """A block that gave up waits for its copies and products before it frees tensor memory and leaves:
    the waits that do not look at the abort flag stand at the end of the warps that start them."""
    code = _code("window_attn.cu")
    body = code[code.index("window_kernel("):]
    waits = [m.start() for m in re.finditer(r"wait_landed\((?!uint|\[)", body)]
    assert len(waits) == 3 and "late_flag, H3B_STATUS" in body
    assert max(waits) < body.index("tmem_dealloc(")
    assert re.search(r"mma_commit\(&drained\[x\]\);\s*__syncwarp\(\);\s*wait_landed\(&drained\[x\], 0\);", body)


def test_last_fills_of_a_ring_are_told_by_its_next_use():
    """The parity that completes with each slot's last fill: that of the ring's next use for the slots before
    it, else the other one, which a slot never filled has passed already.  (A barrier's phases alternate from
    parity 0; a wait for a parity ends when the phase of that parity is not the current one.)"""
    slots = 5
    for fills in range(4 * slots):
        next_slot, parity = fills % slots, fills // slots % 2
        for s in range(slots):
            done = len(range(s, fills, slots))  # fills of the slot
            asked = parity if s < next_slot else parity ^ 1
            waits = [asked == phase % 2 for phase in (done, done - 1)]  # all landed / all but the last
            assert not waits[0], (fills, s)
            if done:
                assert waits[1], (fills, s)


def test_the_query_barrier_of_the_last_item():
    parity = 1
    for fills in range(6):
        assert parity != fills % 2  # landed: the wait is over
        if fills:
            assert parity == (fills - 1) % 2  # under way: it is not
        parity ^= 1
