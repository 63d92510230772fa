"""Bounded waits of the cross-attention kernels, read in their source: a wait that runs out ends for a whole warp at once.

A lane that gave up alone would be missing from the warp's next vote, shuffle or tensor-memory access, and the rest would
wait for it without end, so nothing of this may run on a GPU."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc")


@pytest.mark.parametrize("name,start,end", [
    ("cross_attn.cuh", "} else if (warp == C::kCleanWarp) {", "tmem_dealloc(tmem, C::kTmemCols)"),  # the cleaning and softmax warps
    ("cross_decode.cu", "uint4 qf[KC][NB];", "decode_join<DH, F16>(a, hk"),  # the warps that walk the keys
])
def test_waits_of_whole_warps_have_one_outcome(name, start, end):
    with open(os.path.join(CSRC, name)) as f:
        source = f.read()
    part = source[source.index(start):]
    part = part[:part.index(end)]
    assert re.findall(r"mbar_wait_warp\(", part) and not re.findall(r"mbar_wait\(", part)
