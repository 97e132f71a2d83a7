"""A row's bits and its place among the rows: none of it where the width and all strides are multiples of 8; and rows of such a width at odd strides, which begin at every
place within 16 bytes, against the definition in 64 bits (tolerances of test_block_norm_gpu.py)."""
import pytest
import torch

from test_block_norm_gpu import check, inputs, reference

pytestmark = pytest.mark.gpu


def strided(rows, d, stride, like, fill=777.0):
    store = torch.full((rows * stride + 8,), fill, dtype=like.dtype, device="cuda")
    view = store[:rows * stride].view(rows, stride)[:, :d]
    return store, view


@pytest.mark.parametrize("d,stride,offset", [(1000, 1008, 0), (4096, 4104, 0), (64, 72, 0), (512, 1024, 0), (2048, 2056, 0), (1000, 1008, 3)])
@pytest.mark.parametrize("kind", [0, 1])
def test_equal_rows_at_strides_that_are_multiples_of_8(pkg, torch_cuda, d, stride, offset, kind):
    rows = 700
    one = inputs(1, d, torch.float16, torch.float16, True, d)
    bp = pkg.block_norm_params(d, kind=kind, post=True, gate=pkg.GATE_SIGMOID, gate_rows=True, x_stride=stride, y_stride=stride, out_stride=stride, h_stride=stride, gate_stride=stride)
    got = []
    for n in (1, 7, rows):
        stores = [torch.full((n * stride + 16,), 777.0, dtype=torch.float16, device="cuda")[offset:] for _ in range(5)]
        x, y, g, out, h = (s[:n * stride].view(n, stride)[:, :d] for s in stores)
        x.copy_(one[0].expand(n, d)), y.copy_(one[1].expand(n, d)), g.copy_(one[2].expand(n, d))
        pkg.block_norm(x, y, out, h, n, bp, g, *one[3:])
        torch.cuda.synchronize()
        got.append((out.clone(), h.clone()))
    for out, h in got:
        assert torch.equal(out, got[0][0].expand_as(out)) and torch.equal(h, got[0][1].expand_as(h))


@pytest.mark.parametrize("d,stride", [(1000, 1001), (4096, 4097), (64, 65), (8, 9), (16, 19), (504, 507), (512, 517), (2048, 2051), (6144, 6149), (12000, 12001), (20000, 20003), (32768, 32769)])
@pytest.mark.parametrize("x_bits,y_bits", [(16, 16), (32, 16), (32, 32)])
@pytest.mark.parametrize("rows", [3, 19, 400])
def test_widths_of_whole_chunks_at_odd_strides(pkg, torch_cuda, d, stride, x_bits, y_bits, rows):
    (xt, xk), (yt, yk) = ((torch.float16, pkg.F16) if b == 16 else (torch.float32, pkg.F32) for b in (x_bits, y_bits))
    x0, y0, g0, *w = inputs(rows, d, xt, yt, True, d + rows)
    (_, x), (_, y), (_, g), (so, out), (sh, h) = (strided(rows, d, stride, t) for t in (x0, y0, g0, x0, g0))
    x.copy_(x0), y.copy_(y0), g.copy_(g0)
    bp = pkg.block_norm_params(d, kind=rows % 2, post=True, gate=pkg.GATE_PLAIN, gate_rows=True, x_dtype=xk, y_dtype=yk,
                               x_stride=stride, y_stride=stride, out_stride=stride, h_stride=stride, gate_stride=stride)
    r, tr, hr, th = reference(pkg, bp, x0, y0, g0, *w)
    pkg.block_norm(x, y, out, h, rows, bp, g, *w)
    torch.cuda.synchronize()
    check(out, r, tr, "x_out")
    check(h, hr, th, "h")
    for store, view in ((so, out), (sh, h)):
        view.fill_(777.0)
        assert torch.all(store == 777)
