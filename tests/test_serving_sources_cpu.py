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


def kernels(text):
    """(name, what stands before its wait) of every kernel of a source."""
    for part in text.split("__global__")[1:]:
        body = part[part.index("{", part.index(")", part.index("_kernel("))):]
        yield re.search(r"(\w+_kernel)\(", part).group(1), body[:body.index("pdl_wait();")]


def without_lambdas(text):
    """The names of the lambdas of a text, and the text without their bodies."""
    names = []
    while True:
        m = re.search(r"\bauto (\w+) = \[[^\]]*\]", text)
        if not m:
            return names, text
        names.append(m.group(1))
        at = text.index("{", m.end())
        depth, end = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        text = text[:m.start()] + text[end:]


# What reads or writes memory that the kernel ahead may still be at: elements and targets of pointers that came as arguments, copies, loads and stores, and the helpers that have them.
TOUCHES = re.compile(r"\b(a|p|names|names\.p|a\.p)\.\w+(\.\w+)?\s*\[|\*\s*(a|p|names)\.|\bld\.|\bst\.|\bcp\.async|tma_load|tma_store|\basm\b|atomic\w+|load8|store8|element\(|prefetch_l2|seqs\[|report\(|rename\(|move\(|\.find\(")


def test_nothing_is_touched_before_the_wait():
    """Kernels are launched while the one ahead of them may still run: what stands before the wait is barriers, tensor memory and descriptors."""
    found = 0
    for name in ("block_norm.cu", "proj_w4_sm100.cu", "proj_w4_tc_sm100.cu", "pages.cu"):
        for kernel, before in kernels(source(name)):
            lambdas, plain = without_lambdas(before)
            assert not TOUCHES.search(plain), (kernel, TOUCHES.search(plain).group(0))
            for called in lambdas:
                assert not re.search(rf"\b{called}\(", plain), (kernel, called)
            found += 1
    assert found == 8


def test_the_check_finds_what_it_looks_for():
    ahead = "int x = {};\n pdl_wait();"
    for touch in ("a.refs[3]", "p.kv_len[b]", "*a.count", "a.p.pages[at]", "seqs[i]", "load8(r, row)", 'asm volatile("ld.global.b32 %0;")', "tma_load_2d(s, &map, bar, 0, 0)"):
        assert TOUCHES.search(ahead.format(touch)), touch
    assert without_lambdas("auto f = [&](int i) { if (i) { a.x[i]; } }; int y;")[0] == ["f"]
