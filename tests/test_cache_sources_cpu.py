"""Orders of steps in the cache kernels that no run can show without risk to the GPU, read from their sources."""

from __future__ import annotations

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse_kv_reads_b200", "csrc")


def kernel_body(file: str, name: str) -> str:
    """The text of one kernel, without comments."""
    text = open(os.path.join(CSRC, file)).read()
    text = re.sub(r"//[^\n]*", "", text[text.index(f"\n{name}("):])
    return text[:text.index("\n}\n")]


def test_tensor_memory_is_asked_for_behind_the_wait_for_earlier_launches():
    """An allocation blocks without a limit: a launch that has started early and holds tensor memory while it waits for one
    that has still to allocate would never end."""
    body = kernel_body("skv_attend_prefix.cu", "prefix_mma_kernel")
    assert body.count("tmem_alloc(") == 1 and 0 <= body.index("pdl_wait();") < body.index("tmem_alloc(")


def test_sums_of_the_other_slot_are_read_behind_a_fence_behind_the_barrier():
    """A warp that folds the two slots reads sums whose products another warp has waited for: fence, barrier, fence."""
    body = kernel_body("skv_attend_prefix.cu", "prefix_mma_kernel")
    tail = body[body.index("b_done + 8 * w, 0"):]
    steps = [tail.index(x) for x in ("tcgen05_before_sync();", "bar.sync 1, 256;")]
    fence = tail.find("tcgen05_after_sync();", steps[1])
    assert steps[0] < steps[1] < fence < tail.index("tmem_ld32(")


def test_a_warp_allocates_tensor_memory_together():
    """The allocation is an instruction of a whole warp, whose lanes the loads of the last rows ahead of it may have parted."""
    body = kernel_body("skv_attend_prefix.cu", "prefix_mma_kernel")
    ahead = body[:body.index("tmem_alloc(")]
    assert ahead.rstrip().endswith("__syncwarp();")
