"""Projections with weights of 4 bits against the definition in 64 bits.

Tolerance, with S = sum over the groups of scale * sum |x| (code + zero), as products with codes and with zeros are summed apart: a product is exact (11 bits times
at most 8); a group's sum of G products in fp32, where the tensor cores may cut instead of rounding, is off by (G + 4) 2^-23 of its magnitudes, adding the scaled
groups, warps and blocks by 2^-24 each: groups + 70 of them at most; then the result is rounded, 2^-11 (2^-25 at the bottom) of fp16, 2^-24 of fp32."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(rows, d_in, d_out, group, zeros, seed, top_zero=16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (d_out, d_in // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = ((0.5 + torch.rand(d_in // group, d_out, generator=gen, device="cuda")) * d_in ** -0.5 / 4).half()
    z = torch.randint(0, top_zero, (d_in // group, d_out), generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
    return torch.randn(rows, d_in, generator=gen, device="cuda").half(), codes, scales, z


def reference(X, codes, scales, zeros, out_dtype):
    group = 2 * codes.shape[1] // scales.shape[0]
    q = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1, group).double()
    w = q - (8 if zeros is None else zeros.t().double().unsqueeze(-1))
    s = scales.t().double().unsqueeze(-1)
    W = (w * s).reshape(codes.shape[0], -1)
    ref, size = X.double() @ W.t(), X.double().abs() @ ((2 * q - w) * s).reshape(codes.shape[0], -1).t()
    tol = ((group + 4) * 2.0 ** -23 + (scales.shape[0] + 70) * 2.0 ** -24) * size
    return ref, tol + (2.0 ** -11 * ref.abs() + 2.0 ** -25 if out_dtype == torch.float16 else 2.0 ** -24 * ref.abs())


def check(got, ref, tol):
    assert torch.isfinite(got).all()
    worst = ((got.double() - ref).abs() / tol).max().item()
    assert worst <= 1, f"{worst:.2f} times the tolerance"


def project(pkg, X, codes, scales, zeros, out_dtype=torch.float16):
    out = torch.full((X.shape[0], codes.shape[0]), 777.0, dtype=out_dtype, device="cuda")
    pkg.project_w4(X, pkg.w4_weight(codes, scales, zeros), out, X.shape[0])
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("rows", [1, 2, 5, 8, 9, 16, 17, 24, 31, 32, 33, 48, 63, 64, 65, 130])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_rows(pkg, torch_cuda, rows, group, zeros):
    a = make(rows, 1152, 200, group, zeros, rows)
    check(project(pkg, *a), *reference(*a, torch.float16))


# Lengths of the sum: one group, not a multiple of 128, fewer units than warps, many; widths: one channel, odd ones, below and above a tile.
@pytest.mark.parametrize("d_in,d_out,group", [(32, 1, 32), (32, 8, 32), (64, 33, 64), (96, 7, 32), (128, 64, 128), (160, 31, 32), (192, 65, 64), (224, 129, 32), (384, 16, 128), (1056, 100, 32),
                                              (1088, 257, 64), (4096, 1003, 128), (4096, 4096, 64), (16384, 40, 128), (16384, 1, 64), (8192, 2500, 32)])
@pytest.mark.parametrize("rows", [1, 7, 13, 64])
@pytest.mark.parametrize("zeros", [False, True])
def test_sizes(pkg, torch_cuda, d_in, d_out, group, rows, zeros):
    for dtype in (torch.float16, torch.float32):
        a = make(rows, d_in, d_out, group, zeros, d_in + d_out)
        check(project(pkg, *a, dtype), *reference(*a, dtype))


def test_every_code_and_zero(pkg, torch_cuda):
    """X picks one k at a time: the values of all codes under all zero points, exactly."""
    for group in (32, 64, 128):
        d_in, d_out = 2 * group, 256
        codes = torch.randint(0, 256, (d_out, d_in // 2), device="cuda", dtype=torch.uint8)
        zeros = torch.arange(256, device="cuda", dtype=torch.uint8).repeat(2, 1)             # more than four bits are taken as they are
        scales = torch.ones(2, d_out, dtype=torch.float16, device="cuda")
        q = torch.stack([codes & 15, codes >> 4], -1).reshape(d_out, d_in).float()
        for k in range(0, d_in, 64):
            X = torch.eye(d_in, dtype=torch.float16, device="cuda")[k:k + 64].contiguous()
            assert torch.equal(project(pkg, X, codes, scales, zeros, torch.float32), (q - zeros[0, :, None].float()).t()[k:k + 64])
            assert torch.equal(project(pkg, X, codes, scales, None, torch.float32), (q - 8).t()[k:k + 64])


def test_shards_of_a_larger_matrix(pkg, torch_cuda):
    """Rows and columns of a matrix as they lie in it; strides of X and out; what lies around out stays."""
    X, codes, scales, zeros = make(11, 512, 96, 64, True, 5)
    for k0, k1, n0, n1 in ((0, 256, 0, 96), (128, 512, 16, 80), (64, 128, 3, 4), (384, 512, 95, 96)):
        part = (codes[n0:n1, k0 // 2:k1 // 2], scales[k0 // 64:k1 // 64, n0:n1], zeros[k0 // 64:k1 // 64, n0:n1])
        store = torch.full((13, 100), 777.0, dtype=torch.float32, device="cuda")
        pkg.project_w4(X[:, k0:k1], pkg.w4_weight(*part), store[1:12, 2:], 11, x_stride=512, out_stride=100)
        check(store[1:12, 2:2 + n1 - n0].clone(), *reference(X[:, k0:k1], *(p.contiguous() for p in part), torch.float32))
        store[1:12, 2:2 + n1 - n0] = 777
        assert torch.all(store == 777)


@pytest.mark.parametrize("rows", [1, 16, 64])
def test_a_row_has_no_part_in_others(pkg, torch_cuda, rows):
    X, codes, scales, zeros = make(rows, 1024, 300, 128, True, 6)
    clean = project(pkg, X, codes, scales, zeros)
    X[rows - 1, 5] = float("nan")
    got = project(pkg, X, codes, scales, zeros)
    assert torch.isnan(got[-1]).all() and torch.equal(got[:-1], clean[:-1])
    X[rows - 1, 5] = float("inf")
    got = project(pkg, X, codes, scales, None)
    assert not torch.isfinite(got[-1]).any() and torch.isfinite(got[:-1]).all()


def test_large_results_become_infinite_and_small_ones_are_kept(pkg, torch_cuda):
    X = torch.full((2, 128), 60000.0, dtype=torch.float16, device="cuda")
    codes = torch.full((8, 64), 0xFF, dtype=torch.uint8, device="cuda")
    scales = torch.ones(1, 8, dtype=torch.float16, device="cuda")
    assert torch.all(project(pkg, X, codes, scales, None) == float("inf"))
    assert torch.all(project(pkg, X, codes, scales, None, torch.float32) == 60000 * 7 * 128)
    X.fill_(2.0 ** -24), scales.fill_(2.0 ** -24)
    assert torch.all(project(pkg, X, codes, scales, None, torch.float32) == 7 * 128 * 2.0 ** -48)


def test_equal_calls_give_equal_bits_and_go_where_they_are_sent(pkg, torch_cuda):
    a = make(16, 4096, 1000, 64, True, 7)
    want = project(pkg, *a)
    w, out = pkg.w4_weight(*a[1:]), torch.zeros_like(want)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            pkg.project_w4(a[0], w, out, 16, stream=side)
    for _ in range(5):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    with pytest.raises(pkg.EfaError, match="memory of the host"):
        pkg.project_w4(a[0].cpu(), w, out, 16)


def test_no_rows(pkg, torch_cuda):
    X, codes, scales, zeros = make(1, 128, 8, 128, False, 8)
    out = torch.full((1, 8), 777.0, dtype=torch.float16, device="cuda")
    pkg.project_w4(X, pkg.w4_weight(codes, scales), out, 0)
    torch.cuda.synchronize()
    assert torch.all(out == 777)


def test_many_rows(pkg, torch_cuda):
    """As many rows as there may be, on both ways."""
    a = make(1 << 19, 32, 8, 32, True, 9)
    out = project(pkg, *a)
    for at in (slice(0, 1000), slice((1 << 18) - 500, (1 << 18) + 500), slice((1 << 19) - 1000, 1 << 19)):
        check(out[at], *reference(a[0][at], *a[1:], torch.float16))
    a = make(5000, 1024, 2000, 128, False, 9)
    check(project(pkg, *a), *reference(*a, torch.float16))


def test_a_kind_of_kernel_that_is_first_met_in_a_capture(pkg, torch_cuda):
    """In a process of its own: one call outside of a capture, then every kind of kernel for the first time within one."""
    import subprocess
    import sys
    code = """
import sys; sys.path[:0] = ["tests", "."]
import torch, __graft_entry__ as e
from test_w4_gpu import make, reference, check
pkg = e.load_package()
X, *w = make(1, 128, 64, 128, False, 1)
out = torch.zeros(1, 64, dtype=torch.float16, device="cuda")
pkg.project_w4(X, pkg.w4_weight(*w), out, 1)
cases = [make(r, 2048, 4096, g, True, r + g) for r in (3, 16, 40, 64) for g in (32, 64, 128)] + [make(r, 4096, 6144, 64, False, r) for r in (12, 30)]
outs = [torch.zeros(a[0].shape[0], a[1].shape[0], dtype=torch.float16, device="cuda") for a in cases]
side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
weights = [pkg.w4_weight(*a[1:]) for a in cases]
with torch.cuda.graph(graph, stream=side):
    for a, w, out in zip(cases, weights, outs):
        pkg.project_w4(a[0], w, out, a[0].shape[0], stream=side)
graph.replay()
torch.cuda.synchronize()
for a, out in zip(cases, outs):
    check(out, *reference(*a, torch.float16))
"""
    import conftest
    r = subprocess.run([sys.executable, "-c", code], cwd=conftest.ROOT, capture_output=True, text=True, timeout=200)
    assert r.returncode == 0, r.stderr[-2000:]


def test_calls_on_two_streams_at_a_time(pkg, torch_cuda):
    """Kernels that hold an SM's tensor memory, and others, side by side on one GPU."""
    cases = [make(64, 4096, 4096, 128, True, 1), make(12, 4096, 6144, 64, False, 2), make(1, 8192, 1024, 128, False, 3), make(40, 2048, 4096, 32, True, 4)]
    want = [project(pkg, *a) for a in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    weights, outs = [pkg.w4_weight(*a[1:]) for a in cases], [torch.zeros_like(w) for w in want]
    for _ in range(50):
        for a, w, out, s in zip(cases, weights, outs, streams):
            pkg.project_w4(a[0], w, out, a[0].shape[0], stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, outs)) and pkg.kernel_status()[0] == 0


# More tiles of 32 channels than blocks, by one or by many, whole ones and not; fewer units of k than warps, as many, and more; rows of which little and much is copied.
@pytest.mark.parametrize("d_in,d_out,group", [(32, 9473, 32), (96, 40001, 32), (1024, 9504, 64), (2080, 12001, 32), (4096, 19000, 128), (8256, 9500, 64), (12288, 9985, 128)])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 8])
def test_blocks_that_go_on_to_another_tile(pkg, torch_cuda, d_in, d_out, group, rows):
    a = make(rows, d_in, d_out, group, rows % 2 == 1, d_in + rows)
    out = project(pkg, *a)
    check(out, *reference(*a, torch.float16))
    for _ in range(3):
        assert torch.equal(project(pkg, *a), out)
    assert pkg.kernel_status()[0] == 0


@pytest.mark.parametrize("rows", [4, 16, 32])
def test_an_infinite_scale_is_its_channels_own(pkg, torch_cuda, rows):
    """Also in the last group, behind which a step has none."""
    X, codes, scales, _ = make(rows, 1056, 16200, 32, False, 10)
    clean = project(pkg, X, codes, scales, None)
    scales[32, 5], scales[0, 700] = float("inf"), float("inf")
    got = project(pkg, X, codes, scales, None)
    assert torch.isinf(got[:, [5, 700]]).all()
    rest = [n for n in range(16200) if n not in (5, 700)]
    assert torch.equal(got[:, rest], clean[:, rest])


@pytest.mark.parametrize("rows", [9, 16, 17, 32, 33, 64, 80])
@pytest.mark.parametrize("d_in,group", [(1120, 32), (1088, 64), (1152, 128)])
@pytest.mark.parametrize("d_out,zeros", [(15503, True), (16000, False)])
def test_tiles_that_hold_their_sums_in_tensor_memory(pkg, torch_cuda, rows, d_in, group, d_out, zeros):
    """Every width of these tiles with every group; lengths that end inside a unit of 128."""
    for dtype in (torch.float16, torch.float32):
        a = make(rows, d_in, d_out, group, zeros, rows + d_in)
        check(project(pkg, *a, dtype), *reference(*a, dtype))
    assert pkg.kernel_status()[0] == 0


def test_blocks_of_several_tiles_in_graphs_side_by_side(pkg, torch_cuda):
    """Blocks that stay on their SM for several tiles, two of them and one on tcgen05 at a time, replayed."""
    cases = [make(1, 2048, 16384, 64, True, 1), make(2, 8192, 12000, 128, False, 2), make(48, 2048, 16384, 128, False, 3)]
    want = [project(pkg, *a) for a in cases]
    weights, outs, graphs = [pkg.w4_weight(*a[1:]) for a in cases], [torch.zeros_like(w) for w in want], []
    streams = [torch.cuda.Stream() for _ in cases]
    for a, w, out, s in zip(cases, weights, outs, streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            for _ in range(5):
                pkg.project_w4(a[0], w, out, a[0].shape[0], stream=s)
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, outs)) and pkg.kernel_status()[0] == 0
    del graphs
