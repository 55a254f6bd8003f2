"""What must hold of the decoder kernels' waits and cannot be shown by running them, since it matters when a wait runs out: read from
the sources."""
import os
import re

import pytest

from juliavision_b200 import build

KERNELS = ["cache8_attention.cu", "cache8_prompt.cu", "linear4.cu"]
WAIT = r"\bmbar_\w*wait\w*\("


def source(name):
    with open(os.path.join(build.CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", KERNELS)
def test_a_warp_leaves_a_wait_as_one(name):
    """Every bounded wait is voted on by the whole warp: a lane that gave up alone would leave the others waiting for it in the next vote
    or barrier of the warp, without a limit."""
    text, found = source(name), 0
    while (at := text.find("__all_sync(0xffffffffu,")) >= 0:      # the vote and what stands in its brackets, taken out
        end, depth = text.index("(", at) + 1, 1
        while depth:
            depth += {"(": 1, ")": -1}.get(text[end], 0)
            end += 1
        found += len(re.findall(WAIT, text[at:end]))
        text = text[:at] + text[end:]
    assert found and not re.findall(WAIT, text)


def test_a_stage_is_asked_for_behind_the_reads_of_it():
    """The bulk copies into a stage that a warp has just read are asked for behind a barrier of the warp, which orders its lanes' reads;
    the vote on a wait orders none."""
    text = source("linear4.cu")
    loop = text[text.index("for (int at = 0; at < tiles; ++at)"):]
    loop = loop[:loop.index("fetch();")]
    assert loop.rstrip().endswith("__syncwarp();")
