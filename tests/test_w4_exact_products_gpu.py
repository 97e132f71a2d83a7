"""Projections with 4-bit weights against the definition in 64 bits, with the tolerance of exact products.

code - zero is exact before it is multiplied, and a product of 11 bits and 8 is exact in fp32. With S = sum over the groups of scale * sum |x| |code - zero|: a group's sum of
G products in fp32, where the tensor cores may cut instead of rounding, is off by (G + 4) 2^-23 of its magnitudes; the scaled groups, warps and blocks are added with 2^-24 each,
groups + 70 of them at most; then the result is rounded, 2^-11 (2^-25 at the bottom) of fp16, 2^-24 of fp32. Magnitudes of codes and of zeros by themselves have no part in it."""
import pytest
import torch

from test_w4_gpu import make, project

pytestmark = pytest.mark.gpu


def check(got, ref, tol):
    """Off by no more than the tolerance, which is nothing where all weights are."""
    assert torch.isfinite(got).all()
    off = (got.double() - ref).abs() - tol
    assert (off <= 0).all(), f"{off.max().item():.3g} beyond the tolerance"


def reference(X, codes, scales, zeros, out_dtype):
    group = 2 * codes.shape[1] // scales.shape[0]
    q = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1, group).double()
    W = ((q - (8 if zeros is None else zeros.t().double().unsqueeze(-1))) * scales.t().double().unsqueeze(-1)).reshape(codes.shape[0], -1)
    ref, size = X.double() @ W.t(), X.double().abs() @ W.abs().t()
    tol = ((group + 4) * 2.0 ** -23 + (scales.shape[0] + 70) * 2.0 ** -24) * size
    return ref, tol + (2.0 ** -11 * ref.abs() + 2.0 ** -25 if out_dtype == torch.float16 else 2.0 ** -24 * ref.abs())


# Few rows on mma.sync, blocks that go on, clusters that share k, tcgen05 with all its widths; lengths that end inside a unit.
@pytest.mark.parametrize("d_in,d_out", [(96, 33), (1152, 200), (4096, 4096), (2048, 12001), (8192, 1003), (1088, 16500)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 8, 16, 32, 64, 130])
def test_products_are_exact(pkg, torch_cuda, d_in, d_out, group, rows):
    d_in = -(-d_in // group) * group
    for zeros in (True, False):
        a = make(rows, d_in, d_out, group, zeros, d_in + rows)
        for dtype in (torch.float16, torch.float32):
            check(project(pkg, *a, dtype), *reference(*a, dtype))


@pytest.mark.parametrize("rows", [1, 16, 64])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_weights_near_their_zero_points(pkg, torch_cuda, rows, group):
    """Zero points of up to 15 with codes one step away from them, where codes and zeros apart would be 15 times the weights; exact zeros give 0."""
    gen = torch.Generator(device="cuda").manual_seed(rows + group)
    d_in, d_out = 2048, 9001
    X, _, scales, zeros = make(rows, d_in, d_out, group, True, rows)
    zeros = zeros.clamp(1, 14)
    step = torch.randint(-1, 2, (d_out, d_in // group, group), generator=gen, device="cuda")
    step[5:900] = 0
    q = (zeros.t().long().unsqueeze(-1) + step).reshape(d_out, d_in)
    codes = (q[:, 0::2] | q[:, 1::2] << 4).to(torch.uint8)
    for dtype in (torch.float16, torch.float32):
        out = project(pkg, X, codes, scales, zeros, dtype)
        check(out, *reference(X, codes, scales, zeros, dtype))
        assert torch.all(out[:, 5:900] == 0)
