"""The kernels of shared prefixes and drafts start while the one ahead still runs, so they read global memory past L1: by
``__ldcg``, ``fresh`` and ``fresh_index``, cp.async and TMA.  A line that L1 kept from another use of the memory cannot be
made to show, so the sources are read."""
import re

import pytest

from test_early_reads import code_of


@pytest.mark.parametrize("name", ["drafts.cu", "shared_prefix.cu", "shared_prefix.cuh", "shared_prefix_own.cuh", "shared_prefix_tc.cuh"])
def test_nothing_is_read_through_l1(name):
    code = code_of(name)
    assert not re.findall(r"__(?:ldg|ldca|ldcs|ldlu|ldcv)\b", code)
    for load in re.findall(r"\bld\.(?:\w+\.)*global[\w.:]*|\bld\.global[\w.:]*", code):
        assert ".cg" in load, load
    assert not re.findall(r"cp\.async\.ca\b", code)
