"""Loads and stores of TMEM are instructions of a whole warp, undefined where its lanes come one by one. A warp whose lanes
may have parted (rows behind a sample's end, maxima that only some rows take over) has to meet again before each: looked
for in the source, since a kernel that gets it wrong may still work."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-conv_b200", "csrc")
COLLECTIVE = re.compile(r"\b(tmem_ld16|tmem_st16|lt_load32|at_load|tmem_alloc)\(")
MEETS = ("__syncwarp()", "__all_sync(", "__any_sync(", "__syncthreads()", "at_check_offsets(a)")
#: A lane's own branch: on its row, or on its maximum.
PARTS = re.compile(r"\bif \((!?mine|!?grown|bad|tid == 0|lane == 0)\b|\bcontinue;")


def body(lines, at):
    """Lines [at, end] of the loop whose head is lines[at]."""
    depth, end = 0, at
    while True:
        depth += lines[end].count("{") - lines[end].count("}")
        if depth <= 0:
            return end
        end += 1


def unmet(text):
    """Numbers of the lines whose collective access follows a lane's own branch, in its loop's order too, with no meeting between."""
    lines = [line.split("//")[0] for line in text.splitlines()]
    heads = [i for i, line in enumerate(lines) if re.search(r"\bfor \(", line) and "{" in line]
    found = []

    def meets(j):
        """Whether the warp meets there: by itself, or in a wait that asks all lanes."""
        named = [k for k in range(j) if "auto wait = " in lines[k]]
        asks = named and "wait(" in lines[j] and "__all_sync(" in "".join(lines[named[-1]:named[-1] + 3])
        return asks or any(m in lines[j] for m in MEETS)
    for i, line in enumerate(lines):
        if not COLLECTIVE.search(line) or "__device__" in line:
            continue
        for j in range(i - 1, -1, -1):
            if meets(j) or "__device__" in lines[j]:
                break
            # a loop that the access is in: what parts the lanes anywhere in it comes before the access too
            inside = j in heads and body(lines, j) >= i
            if PARTS.search(lines[j]) or (inside and any(PARTS.search(b) for b in lines[j:body(lines, j) + 1])):
                found.append(i + 1)
                break
    return found


@pytest.mark.parametrize("name", ["attention_tc_fwd.cu", "attention_tc_bwd.cu"])
def test_lanes_meet_before_tmem(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    assert COLLECTIVE.search(text)
    assert unmet(text) == []


def test_offsets_check_ends_together():
    with open(os.path.join(CSRC, "attention_common.cuh")) as f:
        text = f.read()
    check = text[text.index("void at_check_offsets("):]
    assert "__syncwarp();" in check[check.index("if (bad)"):check.index("\n}\n")]


def test_the_search_finds_a_parted_warp():
    loop = "for (int c = 0; c < D; c += 16) {\n%s    tmem_ld16(t + c, o);\n    if (!mine) continue;\n    store(o);\n}\n"
    assert unmet(loop % "") == [2] and unmet(loop % "    __syncwarp();\n") == []
    assert unmet("if (grown) top = now;\ntmem_ld16(t, o);\n") == [2]
    assert unmet("if (grown) top = now;\n__syncwarp();\nfor (int c = 0; c < D; c += 16) {\n    tmem_ld16(t + c, o);\n}\n") == []
