"""How the products of 4-bit weights are divided among clusters, on the CPU: never into clusters that the device cannot hold."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT

SOURCE = """
#include "w4_plan.h"
extern "C" void divide(int d_out, int row_tiles, int units, const int* at_once, int* out)
{
    const efa::W4Division to = efa::w4_division(d_out, row_tiles, units, at_once);
    out[0] = to.channels; out[1] = to.parts;
}
"""
B200 = [0, 148, 70, 46, 34, 26, 23, 18, 16]           # one block to an SM, clusters within one part of the GPU


@pytest.fixture(scope="module")
def divide(tmp_path_factory):
    d = tmp_path_factory.mktemp("division")
    (d / "divide.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "eager-flash-attention_b200", "csrc"),
                    str(d / "divide.cpp"), "-o", str(d / "divide.so")], check=True)
    lib = ctypes.CDLL(str(d / "divide.so"))

    def run(d_out, row_tiles, units, at_once):
        out = (ctypes.c_int * 2)()
        lib.divide(d_out, row_tiles, units, (ctypes.c_int * 9)(*at_once), out)
        return tuple(out)
    return run


SIZES = [(d_out, row_tiles, units) for d_out in (1, 200, 256, 257, 1024, 4096, 6144, 16384, 32768, 65536) for row_tiles in (1, 2, 7) for units in (1, 2, 5, 8, 32, 64, 131)]


def test_the_fewest_rounds(divide):
    for d_out, row_tiles, units in SIZES:
        def time(c, p):
            clusters = -(-d_out // (2 * c)) * row_tiles
            return -(-clusters // B200[p]) * (4 + 0.6 * -(-units // p) + (p > 1))
        best = min(time(c, p) for c in (128, 112, 96) for p in range(1, min(8, units) + 1))
        c, p = divide(d_out, row_tiles, units, B200)
        assert c in (128, 112, 96) and 1 <= p <= min(8, units) and time(c, p) <= best * 1.01


@pytest.mark.parametrize("missing", [{8}, {5, 6, 7, 8}, {2, 3, 4, 5, 6, 7, 8}, {3, 7}])
def test_clusters_that_do_not_fit_are_no_choice(divide, missing):
    at_once = [0 if p in missing else n for p, n in enumerate(B200)]
    for size in SIZES:
        assert divide(*size, at_once)[1] not in missing


def test_a_block_by_itself_there_always_is(divide):
    for size in SIZES:
        assert divide(*size, [0] * 9)[1] == 1
