"""CPU check of the kernels' sources: dynamic shared memory begins behind the static one, whose size need not be a multiple
of 16, so an array that is written or read 16 bytes at a time has to ask for its alignment."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-thresholded-attention_amd", "csrc")
FILES = [f for f in sorted(glob.glob(os.path.join(CSRC, "*.hip"))) if "extern __shared__" in open(f).read()]


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_dynamic_shared_arrays_are_16_byte_aligned(path):
    for line in re.findall(r"extern __shared__[^;]*;", open(path).read()):
        assert "__align__(16)" in line, line
