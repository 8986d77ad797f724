"""What the compiler made of the paged cache's kernels that no test of results shows: no register spilled inside a loop of products, and no
private array put into LDS -- its address is made from the dispatch packet, which lies in host memory: 12 us a launch."""

import os
import re

import pytest

from test_k_loop_assembly import CSRC, compile_to_assembly, k_loops


@pytest.mark.parametrize("source", ["paged_attention.hip", "paged_cache.hip"])
def test_assembly(tmp_path, source):
    text = compile_to_assembly(os.path.join(CSRC, source), str(tmp_path / "out.s"))
    assert text.count(".amdhsa_user_sgpr_dispatch_ptr 0") > 0 and ".amdhsa_user_sgpr_dispatch_ptr 1" not in text
    loops = list(k_loops(text))
    assert (len(loops) > 0) == (source == "paged_attention.hip")
    for kernel, loop in loops:
        assert not any("scratch_" in line for line in loop), kernel
    assert all(int(n) <= 48 for n in re.findall(r"; ScratchSize: (\d+)", text))  # (some words outside of the loops)
