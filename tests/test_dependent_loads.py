"""Operators that are launched to overlap the kernel ahead of them read by plain loads what that kernel may have written.

A kernel launched that way is resident while the one ahead still writes.  Non-coherent loads (__ldg, ld.global.nc, const __restrict__) promise
that their data stays as it is for the whole of the kernel, its start included, and may be moved ahead of the wait; no run shows for certain
that one was not.  Lists, places, scales and operands of these operators come from one another.
"""
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "lc0_b200", "csrc")
FILES = ["quantize.cu", "route.cu", "qk_norm.cu", "grouped.cu", "grouped_pair.cu", "grouped_rows.cu", "grouped.cuh", "grouped_tc.cuh", "chunk8.cuh"]


@pytest.mark.parametrize("name", FILES)
def test_no_load_promises_that_its_data_is_constant(name):
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)
    assert not re.findall(r"__ldg\s*\(|ld\.global\.nc|__restrict__|ld\.global[.\w]*\.nc", code)


def test_they_wait_ahead_of_their_loads():
    """Every kernel of these files waits for the one ahead of it."""
    for name in FILES:
        if not name.endswith(".cu"):
            continue
        with open(os.path.join(CSRC, name)) as f:
            kernels = re.split(r"\n__global__ ", f.read())[1:]
        assert kernels, name
        for k in kernels:
            assert "grid_dependency_wait();" in k, (name, k[:120])
