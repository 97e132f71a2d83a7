"""Which kernel the products of 4-bit weights take, and how they are divided among clusters, on the CPU: never into clusters that the device cannot hold."""
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
    out[0] = to.channels; out[1] = to.parts; out[2] = (int)to.rounds; out[3] = to.units;
}
extern "C" int tcgen05(int d_in, int d_out, int rows, int group, const int* at_once)
{
    const efa::W4Division to = efa::w4_division(d_out, (rows + 63) / 64, (d_in + 127) / 128, at_once);
    if (efa::w4_tc_least(d_in, d_out, rows, group) > efa::w4_tc_time(to, d_in, d_out, rows, group)) return -1;
    return efa::w4_tc_time(to, d_in, d_out, rows, group) < efa::w4_mma_time(d_in, d_out, rows, group, 148);
}
"""
B200 = [0, 148, 74, 45, 33, 26, 22, 15, 15]           # one block to an SM, clusters within one part of the GPU


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    d = tmp_path_factory.mktemp("division")
    (d / "divide.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "eager-flash-attention_b200", "csrc"),
                    str(d / "divide.cpp"), "-o", str(d / "divide.so")], check=True)
    return ctypes.CDLL(str(d / "divide.so"))


@pytest.fixture(scope="module")
def divide(library):
    def run(d_out, row_tiles, units, at_once):
        out = (ctypes.c_int * 4)()
        library.divide(d_out, row_tiles, units, (ctypes.c_int * 9)(*at_once), out)
        c, p, rounds, share = out
        assert share == -(-units // p) and rounds == -(-(-(-d_out // (2 * c)) * row_tiles) // max(1, at_once[p]))
        return c, p
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


# (d_in, d_out, group, rows): us on mma.sync, on tcgen05, where they are further apart than the figures are off.
MEASURED = {(1024, 1024, 128, 16): (3.07, 4.91), (4096, 2048, 32, 9): (5.44, 8.16), (16384, 1024, 32, 33): (21.1, 33.9), (16384, 1024, 64, 64): (19.4, 22.6), (8192, 2048, 32, 48): (17.7, 20.9),
            (4096, 4096, 64, 16): (7.14, 9.16), (8192, 1024, 128, 16): (6.37, 8.88), (6144, 2048, 32, 64): (14.1, 17.8), (5120, 1536, 32, 96): (12.4, 16.0),
            (512, 8192, 128, 64): (15.5, 8.5), (512, 8192, 32, 64): (16.1, 9.5), (1536, 5120, 128, 32): (8.98, 7.43), (8192, 2048, 128, 17): (11.5, 9.8), (8192, 8192, 128, 16): (18.0, 14.5),
            (4096, 14336, 64, 12): (17.8, 15.4), (14336, 4096, 128, 9): (19.3, 15.3)}


def test_the_kernel_that_was_measured_to_be_faster(library):
    at_once = (ctypes.c_int * 9)(*B200)
    for size, (mma, tc) in MEASURED.items():
        assert library.tcgen05(size[0], size[1], size[3], size[2], at_once) == (tc < mma), size


def test_the_largest_sizes_are_counted_without_overflow(library):
    at_once = (ctypes.c_int * 9)(*B200)
    for group in (32, 64, 128):
        assert library.tcgen05(1 << 24, 1 << 24, 1 << 19, group, at_once) == 1
        assert library.tcgen05(1 << 24, 1, 9, group, at_once) in (0, 1) and library.tcgen05(group, 1 << 24, 1 << 19, group, at_once) in (0, 1)


def test_the_least_that_tcgen05_takes_is_no_more_than_it_takes(library):
    for at_once in (B200, [0, 148] + [0] * 7, [0] * 9):
        at_once = (ctypes.c_int * 9)(*at_once)
        for group in (32, 64, 128):
            for d_out, _, units in SIZES:
                for rows in (9, 17, 33, 64, 65, 500):
                    assert library.tcgen05(128 * units, d_out, rows, group, at_once) >= 0
