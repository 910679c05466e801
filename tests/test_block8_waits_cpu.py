"""CPU suite: bounded waits of the kernels on tcgen05. A lane of a wait that runs out gives up by its own clock and its own look at what others have given up, so the lanes
of a warp may come back with different answers. Where the warp goes on as a whole (tcgen05.ld, votes, __syncwarp) its lanes have to agree on one (warp_wait); the
form of single lanes (barrier_wait) is for what one elected lane does."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alphasparse_b200", "csrc")
KERNELS = [f for f in sorted(glob.glob(os.path.join(CSRC, "*.cu"))) if "tc::" in open(f).read()]


def waits_outside_elected_lanes(text):
    """Line numbers of calls of barrier_wait that no block behind `if (tc::one_lane())` encloses."""
    text = re.sub(r"//[^\n]*", "", text)
    found, blocks = [], []
    for m in re.finditer(r"[{}]|\bbarrier_wait\b", text):
        if m.group() == "{":
            blocks.append(text[: m.start()].rstrip().endswith("if (tc::one_lane())"))
        elif m.group() == "}":
            blocks.pop()
        elif not any(blocks):
            found.append(text[: m.start()].count("\n") + 1)
    return found


def test_the_search_finds_what_it_should():
    one, warp = "if (tc::one_lane())\n{\n for (;;) { if (!tc::barrier_wait(&b)) goto end; }\n}\n", "for (;;)\n{\n if (!tc::barrier_wait(&b)) goto end;\n}\n"
    assert waits_outside_elected_lanes(one) == [] and waits_outside_elected_lanes(one + warp) == [7] and waits_outside_elected_lanes(warp + one) == [3]
    assert waits_outside_elected_lanes("// barrier_wait\n{ warp_wait(); }") == []


@pytest.mark.parametrize("path", KERNELS, ids=[os.path.basename(f) for f in KERNELS])
def test_warps_that_go_on_as_a_whole_agree_on_their_waits(path):
    assert waits_outside_elected_lanes(open(path).read()) == []
