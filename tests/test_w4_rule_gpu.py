"""Projections with 4-bit weights around the line between their kernels: every width and group of the one on tcgen05, and sizes that go to the other."""
import pytest
import torch

from test_w4_gpu import check, make, project, reference

pytestmark = pytest.mark.gpu


# Wide and short, narrow and long, odd; one row tile, two, three and four, and a second tile of 64.
@pytest.mark.parametrize("d_in,d_out", [(512, 8200), (2048, 12290), (8192, 2049), (1152, 28000), (16384, 1024)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("rows", [9, 16, 24, 40, 64, 70])
def test_both_sides_of_the_line(pkg, torch_cuda, d_in, d_out, group, zeros, rows):
    a = make(rows, d_in, d_out, group, zeros, d_in + rows)
    for dtype in (torch.float16, torch.float32):
        check(project(pkg, *a, dtype), *reference(*a, dtype))
    assert pkg.kernel_status()[0] == 0
