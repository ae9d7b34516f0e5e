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
