"""Kernels that start while the kernel before them ends may not read what it
writes by read-only loads (ld.global.nc, __ldg: constant over the kernel's
life).  No run shows it reliably, so the sources are searched."""
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "lal_b200", "csrc")


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"/\*.*?\*/|//[^\n]*", "", f.read(), flags=re.S)


@pytest.mark.parametrize("name", ["tail_q8.cu", "tail_q4.cu", "tail_layer.h"])
def test_layer_operators_have_no_read_only_loads(name):
    assert not re.search(r"__ldg\b|\.nc\b", code(name))


def test_the_fused_tail_reads_the_hidden_vector_by_ordinary_loads():
    reads = re.findall(r"(\w+)\(\s*(?:h|p\.hidden)\s*\+", code("tail_kernels.cu"))
    assert reads and set(reads) == {"__ldcg"}
