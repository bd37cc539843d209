"""Kernels that are launched while their predecessor still runs (griddepcontrol) may not read through the read-only path, whose
data has to stay unwritten for as long as the kernel is resident: no such load in their sources, and no argument that
the compiler may read that way."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "g1.cu_b200", "csrc")
FILES = [f for f in sorted(os.listdir(CSRC)) if "griddepcontrol.wait" in open(os.path.join(CSRC, f)).read()]


def test_there_are_some():
    assert {"g1_gated.cuh", "g1_opt.cuh"} <= set(FILES)


@pytest.mark.parametrize("name", FILES)
def test_no_read_only_loads(name):
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    for word in ("__ldg", "global.nc", "ldu.global"):
        assert word not in code, word
    assert not re.search(r"const\s+\w+(<[^>]*>)?\s*\*\s*__restrict__", code)
