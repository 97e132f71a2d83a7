"""Norms, 4-bit projections and pages whose rows lie further apart than 32 bits count: strides of gigabytes, and dense tensors of more than 2^31 elements."""
import pytest
import torch

from test_block_norm_gpu import check as check_norm, inputs, reference as norm_reference
from test_w4_gpu import check, make, reference

pytestmark = pytest.mark.gpu


def far(rows, width, stride, dtype):
    """Rows of a tensor, ``stride`` elements apart; what lies between them is not looked at."""
    return torch.empty((rows - 1) * stride + width, dtype=dtype, device="cuda").as_strided((rows, width), (stride, 1))


@pytest.mark.parametrize("d,stride", [(4096, (1 << 30) + 8), (1001, (1 << 30) + 1), (64, (1 << 30) + 3)])
def test_norms_of_rows_gigabytes_apart(pkg, torch_cuda, d, stride):
    rows = 4
    x0, y0, g0, *w = inputs(rows, d, torch.float16, torch.float16, False, d)
    x, h = (far(rows, d, stride, torch.float16) for _ in range(2))
    x.copy_(x0)
    bp = pkg.block_norm_params(d, post=True, gate=pkg.GATE_SIGMOID, x_stride=stride, out_stride=stride, h_stride=stride)
    r, tr, hr, th = norm_reference(pkg, bp, x0, y0, g0, *w)
    pkg.block_norm(x, y0, x, h, rows, bp, g0, *w)
    check_norm(x, r, tr, "x_out")
    check_norm(h, hr, th, "h")


@pytest.mark.parametrize("d", [32768, 2049])
def test_norms_of_more_than_2_31_elements(pkg, torch_cuda, d):
    rows = (1 << 31) // d + 50
    x = torch.randn(64, d, device="cuda").half().repeat(-(-rows // 64), 1)[:rows].contiguous()
    h, bp = torch.empty_like(x), pkg.block_norm_params(d, eps=1e-5)
    pkg.block_norm(x, None, None, h, rows, bp)
    for at in (slice(0, 3), slice(rows - 60, rows)):
        _, _, hr, th = norm_reference(pkg, bp, x[at], None, None, None, None, None, None)
        check_norm(h[at], hr, th, "h")


@pytest.mark.parametrize("rows,d_in,d_out", [(12, 1024, 200), (12, 2048, 16500), (8, 512, 9700)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_projections_of_rows_gigabytes_apart(pkg, torch_cuda, rows, d_in, d_out, dtype):
    stride = (1 << 28) + 8 if rows > 8 else (1 << 29) + 8
    X0, *w = make(rows, d_in, d_out, 64, True, rows)
    X, out = far(rows, d_in, stride, torch.float16), far(rows, d_out, stride, dtype)
    X.copy_(X0)
    pkg.project_w4(X, pkg.w4_weight(*w), out, rows, x_stride=stride, out_stride=stride)
    check(out, *reference(X0, *w, dtype))


@pytest.mark.parametrize("rows", [3, 64])
def test_projections_of_weights_gigabytes_apart(pkg, torch_cuda, rows):
    X, codes0, scales0, zeros0 = make(rows, 4096, 260, 64, True, rows)
    codes, scales, zeros = far(260, 2048, 1 << 25, torch.uint8), far(64, 260, (1 << 26) + 1, torch.float16), far(64, 260, (1 << 26) + 5, torch.uint8)
    for x, y in ((codes, codes0), (scales, scales0), (zeros, zeros0)):
        x.copy_(y)
    out = torch.zeros(rows, 260, dtype=torch.float32, device="cuda")
    pkg.project_w4(X, pkg.w4_weight(codes, scales, zeros), out, rows)
    check(out, *reference(X, codes0, scales0, zeros0, torch.float32))


def test_pages_gigabytes_apart(pkg, torch_cuda):
    stride, shape = (1 << 30) + 64, (4, 2, 16, 16)
    parts = [torch.empty(3 * stride + 512, dtype=torch.float16, device="cuda").as_strided(shape, (stride, 256, 16, 1)) for _ in range(2)]
    want = [torch.randn(shape, device="cuda").half() for _ in range(2)]
    for x, y in zip(parts, want):
        x.copy_(y)
    cache = pkg.paged_cache(*parts)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pkg.pages_copy(cache, ints(3, 0), ints(1, 2))
    refs, pages, kv = ints(0, 0, 0, 1), ints(3, -7, -7, -7).view(2, 2), ints(5, 0)
    pool = pkg.page_pool(refs, pages, kv, 16)
    ws = torch.zeros(pkg.pages_workspace(pool), dtype=torch.uint8, device="cuda")
    pkg.pages_compact(pool, cache, pages, refs, ints(0, 0, 0, 0), ws)              # page 3 to page 0
    for x, y in zip(parts, want):
        assert torch.equal(x, torch.stack([y[3], y[3], y[0], y[3]]))
    assert refs.tolist() == [1, 0, 0, 0] and pages.tolist() == [[0, -7], [-7, -7]]


@pytest.mark.parametrize("d_in,d_out,group,rows", [(1 << 24, 3, 128, 1), (1 << 24, 40, 32, 9), (1 << 23, 300, 64, 17), (32, 1 << 24, 32, 1), (64, (1 << 24) - 5, 64, 9), (128, 1 << 24, 128, 17)])
def test_projections_of_the_longest_and_widest_matrices(pkg, torch_cuda, d_in, d_out, group, rows):
    X, *w = make(rows, d_in, d_out, group, rows != 9, rows)
    out = torch.full((rows, d_out), 777.0, dtype=torch.float32, device="cuda")
    pkg.project_w4(X, pkg.w4_weight(*w), out, rows)
    torch.cuda.synchronize()
    step = max(1, (1 << 26) // d_in)
    for lo in range(0, d_out, max(step, d_out // 8)):                               # slices of the channels, the first and the last among them
        at = slice(lo, min(d_out, lo + step)) if lo + max(step, d_out // 8) < d_out else slice(max(0, d_out - step), d_out)
        part = (w[0][at], w[1][:, at], None if w[2] is None else w[2][:, at])
        check(out[:, at], *reference(X, *(p if p is None else p.contiguous() for p in part), torch.float32))
    assert pkg.kernel_status()[0] == 0
