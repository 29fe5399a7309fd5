"""Waits of the kernels of shared prefixes and drafts whose end a whole warp goes by: a wait that runs out in some lanes only cannot be
made to show, so the sources are read."""
import re

import pytest

from test_early_reads import code_of


@pytest.mark.parametrize("name", ["shared_prefix.cu", "shared_prefix_own.cuh", "shared_prefix_tc.cuh"])
def test_a_wait_ends_for_all_lanes(name):
    """Its verdict is voted on, or one lane's that the others are told; what is only waited for has no verdict."""
    code = re.sub(r"bool wait_bar\(", "", code_of(name))
    waits = list(re.finditer(r"\b(?:wait_bar|mbar_wait(?:<true>)?)\(", code))
    assert waits
    for w in waits:
        line = code[code.rfind("\n", 0, w.start()) + 1:code.find("\n", w.end())]
        voted = "__all_sync(0xffffffffu, " + w[0] in line
        unused = re.search(r"(?:^\s*|\) )" + re.escape(w[0]), line) and line.rstrip().endswith(");")
        told = re.match(r"\s*ok = mbar_wait\(", line) and "__shfl_sync(0xffffffffu, ok, 0)" in code[w.end():w.end() + 900]
        assert voted or unused or told, line


@pytest.mark.parametrize("name, barrier", [("drafts.cu", r"cluster_sync\(\);"), ("shared_prefix.cu", r'asm volatile\("bar\.sync'),
                                           ("shared_prefix_own.cuh", r'asm volatile\("barrier\.cluster\.arrive')])
def test_barriers_of_whole_warps_are_met_as_one(name, barrier):
    """Instructions that want a warp's lanes together stand behind ``__syncwarp``, not behind what single lanes do."""
    code = code_of(name)
    found = list(re.finditer(barrier, code))
    assert found
    for b in found:
        assert code[:b.start()].rstrip().endswith("__syncwarp();"), code[b.start() - 200:b.end()]


@pytest.mark.parametrize("name, behind, instruction", [
    ("shared_prefix_tc.cuh", r"mbar_arrive\(&bars->k_empty", "tmem_ld32"), ("shared_prefix_tc.cuh", r"if \(r >= left\)", "tmem_ld16"),
    ("shared_prefix_tc.cuh", r"if \(live && s == 0\)", "tmem_ld16"),
    ("shared_prefix_own.cuh", r"if \(!\(top > m\[n\]\[e\] \+ kGrowth\)\) continue;", "transposed")])
def test_a_warp_is_one_again_behind_what_some_lanes_do(name, behind, instruction):
    code = code_of(name)
    branch = list(re.finditer(behind, code))
    assert len(branch) == 1
    rest = code[branch[0].end():]
    assert "__syncwarp();" in rest[:rest.index(instruction)]
