"""What the sources of the serving kernels have to say for themselves, on a machine without a GPU."""
import os
import re

from conftest import ROOT

CSRC = os.path.join(ROOT, "eager-flash-attention_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_the_table_of_scales_is_ordered_between_lanes():
    """Written by one lane, read by others: a __syncwarp between the last write and the first read, and between the reads and the next unit's writes. Votes and the
    barrier of the copies order nothing of it."""
    body = source("proj_w4_sm100.cu")
    loop = body[body.index("auto tile = [&]()"):body.index("auto put = ")]
    write, read = loop.index("tabulate();"), loop.index("= table[")
    assert "__syncwarp();" in loop[write:read]
    assert "__syncwarp();" in loop[loop.rindex("= table["):]
