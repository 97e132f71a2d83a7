"""Norms before and after a block with its gate and residual addition, against the definition in 64 bits.

Tolerances, with u = 2^-24: everything is fp32 until it is stored. A sum over a row is a chain of at most 32 elements in a thread and a tree of ten levels,
off by 42 u of the sum of magnitudes, which leaves 21 u (and rsqrtf's 2^-22) of a norm's scale; a mean is off by 42 u of the mean magnitude. A sigmoid takes exp
with 2 + 1.16 |g| units in the last place: 18 u with |g| up to 8, and a quotient. So n and r are off by at most 64 u of A, the magnitudes that are
added up in them, where a layer norm's v counts as |v| + mean |v|. The second norm sees that error as an error of its input, of its mean and of its
scale (relative: that of rms A to rms v) next to its own. Last, a rounding: half a step, 2^-11 (2^-25 at the bottom) of fp16, 2^-24 of fp32."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def normed(v, A, kind, eps, w, b):
    """norm(v) in fp64 and the magnitude that 128 u of it is off by at most, where v is off by 64 u A."""
    d = v.shape[-1]
    c = v - v.sum(-1, keepdim=True) / d if kind else v
    ms = (c * c).sum(-1, keepdim=True) / d + eps
    scale = 1 / torch.sqrt(ms)
    size = A + (A.mean(-1, keepdim=True) if kind else 0)
    size = scale * (size + c.abs() * (1 + scale * (size * size).mean(-1, keepdim=True).sqrt()))
    out = c * scale
    if w is not None:
        out, size = out * w.double(), size * w.double().abs()
    if b is not None:
        out, size = out + b.double(), size + b.double().abs()
    return out, size


def rounded(v, dtype):
    return 2.0 ** -11 * v.abs() + 2.0 ** -25 if dtype == torch.float16 else U * v.abs() + 2.0 ** -149


def reference(pkg, bp, x, y, gate, post_w, post_b, pre_w, pre_b):
    """(x_out, tolerance, h, tolerance) in fp64."""
    r = A = 0
    if y is not None:
        n, A = y.double(), y.double().abs()
        if bp.post:
            n, A = normed(n, A, bp.kind, bp.eps, post_w, post_b)
            A = A * 2
        if gate is not None:
            g = gate.double()
            g = 1 / (1 + torch.exp(-g)) if bp.gate == pkg.GATE_SIGMOID else g
            n, A = n * g, A * g.abs()
        r, A = bp.block_scale * n, abs(bp.block_scale) * A
    if x is not None:
        r, A = r + bp.residual_scale * x.double(), A + (bp.residual_scale * x.double()).abs()
    x_dtype = torch.float16 if bp.x_dtype == pkg.F16 else torch.float32
    h, size = normed(r, A, bp.kind, bp.eps, pre_w, pre_b)
    return r, 64 * U * A + rounded(r, x_dtype), h, 128 * U * size + rounded(h, torch.float16)


def check(got, ref, tol, what):
    assert torch.isfinite(got).all(), what
    worst = ((got.double() - ref).abs() / tol).max().item()
    assert worst <= 1, f"{what}: {worst:.2f} times the tolerance"


def inputs(rows, d, x_dtype, y_dtype, gate_rows, seed, mean=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    x, y = (3 * normal(rows, d) + mean).to(x_dtype), (normal(rows, d) + mean).to(y_dtype)
    gate = normal(rows if gate_rows else 1, d).clamp(-8, 8).half()
    w = [(1 + 0.2 * normal(d)).half() for _ in range(2)] + [(0.1 * normal(d)).half() for _ in range(2)]
    return x, y, gate, w[0], w[2], w[1], w[3]


def types(pkg, bits):
    return (torch.float16, pkg.F16) if bits == 16 else (torch.float32, pkg.F32)


def run(pkg, bp, rows, x, y, gate, post_w, post_b, pre_w, pre_b, x_dtype=None):
    d = bp.d
    x_out = torch.full((rows, d), 777.0, dtype=torch.float16 if bp.x_dtype == pkg.F16 else torch.float32, device="cuda")
    h = torch.full((rows, d), 777.0, dtype=torch.float16, device="cuda")
    pkg.block_norm(x, y, x_out, h, rows, bp, gate, post_w, post_b, pre_w, pre_b)
    torch.cuda.synchronize()
    return x_out, h


@pytest.mark.parametrize("rows", [1, 2, 5, 9, 40])
@pytest.mark.parametrize("d", [1, 3, 9, 57, 58, 63, 65, 121, 122, 249, 250, 505, 506, 1017, 1018, 2041, 2042, 4089, 4090])
def test_odd_widths(pkg, torch_cuda, d, rows):
    """Rows at every place within 16 bytes, at and behind the widths where the kernels change."""
    for x_bits, y_bits in ((16, 16), (32, 16), (32, 32)):
        (xt, xk), (yt, yk) = types(pkg, x_bits), types(pkg, y_bits)
        x, y, gate, *w = inputs(rows, d, xt, yt, rows > 2, d + rows)
        bp = pkg.block_norm_params(d, kind=rows % 2, eps=1e-5, post=True, gate=pkg.GATE_PLAIN, gate_rows=rows > 2, residual_scale=0.75, block_scale=0.5, x_dtype=xk, y_dtype=yk)
        r, tr, h, th = reference(pkg, bp, x, y, gate, *w)
        got_r, got_h = run(pkg, bp, rows, x, y, gate, *w)
        check(got_r, r, tr, "x_out")
        check(got_h, h, th, "h")


# Widths: one element, below, at and above the 256 a warp's chunk has, above 512, 1024 and what a block takes with one, two and four chunks, odd ones.
@pytest.mark.parametrize("d", [1, 2, 7, 8, 31, 64, 100, 255, 256, 264, 513, 1000, 1024, 1025, 1032, 2049, 4096, 4104, 5001, 8192, 16384, 16392, 20001, 32768])
@pytest.mark.parametrize("kind", [0, 1])
def test_widths(pkg, torch_cuda, d, kind):
    rows = 5 if d > 4096 else 37
    x, y, gate, *w = inputs(rows, d, torch.float16, torch.float16, False, d)
    bp = pkg.block_norm_params(d, kind=kind, eps=1e-5, post=True, gate=pkg.GATE_SIGMOID, residual_scale=0.75, block_scale=0.5)
    r, tr, h, th = reference(pkg, bp, x, y, gate, *w)
    got_r, got_h = run(pkg, bp, rows, x, y, gate, *w)
    check(got_r, r, tr, "x_out")
    check(got_h, h, th, "h")


@pytest.mark.parametrize("x_bits,y_bits", list(itertools.product((16, 32), (16, 32))))
@pytest.mark.parametrize("kind,post,gate,gate_rows,biases", [(0, True, 1, True, False), (0, False, 2, True, False), (1, True, 2, False, True), (1, False, 0, False, True),
                                                             (0, True, 0, False, True), (1, True, 1, False, False)])
@pytest.mark.parametrize("d", [96, 1048, 1337])
def test_kinds_and_types(pkg, torch_cuda, d, x_bits, y_bits, kind, post, gate, gate_rows, biases):
    (xt, xk), (yt, yk) = types(pkg, x_bits), types(pkg, y_bits)
    rows = 19
    x, y, g, post_w, post_b, pre_w, pre_b = inputs(rows, d, xt, yt, gate_rows, d + x_bits)
    g = g if gate else None
    post_b, pre_b = (post_b, pre_b) if biases else (None, None)
    post_w = post_w if post else None
    bp = pkg.block_norm_params(d, kind=kind, post=post, gate=gate, gate_rows=gate_rows, residual_scale=1.0, block_scale=-0.25, x_dtype=xk, y_dtype=yk)
    r, tr, h, th = reference(pkg, bp, x, y, g, post_w, post_b, pre_w, pre_b)
    got_r, got_h = run(pkg, bp, rows, x, y, g, post_w, post_b, pre_w, pre_b)
    check(got_r, r, tr, "x_out")
    check(got_h, h, th, "h")


def test_a_mean_far_above_the_spread(pkg, torch_cuda):
    """Values around 64 with a spread of a sixteenth: squares less the mean's square would have lost it."""
    for d in (512, 4096):
        x, y, g, *w = inputs(9, d, torch.float32, torch.float32, False, 1)
        x, y = 64 + x / 48, 64 + y / 16
        bp = pkg.block_norm_params(d, kind=pkg.NORM_LAYER, post=True, x_dtype=pkg.F32, y_dtype=pkg.F32)
        r, tr, h, th = reference(pkg, bp, x, y, None, *w)
        got_r, got_h = run(pkg, bp, 9, x, y, None, *w)
        check(got_r, r, tr, "x_out")
        check(got_h, h, th, "h")


@pytest.mark.parametrize("d", [64, 4096, 2049])
def test_parts_that_are_left_out(pkg, torch_cuda, d):
    x, y, g, post_w, post_b, pre_w, pre_b = inputs(6, d, torch.float16, torch.float16, False, 2)
    before = pkg.block_norm_params(d, eps=1e-5, residual_scale=0.5)          # the norm before the first block
    r, tr, h, th = reference(pkg, before, x, None, None, None, None, pre_w, None)
    got_r, got_h = run(pkg, before, 6, x, None, None, None, None, pre_w, None)
    check(got_r, r, tr, "x_out")
    check(got_h, h, th, "h")
    pkg.block_norm(x, None, None, got_h.zero_(), 6, before, pre_w=pre_w)     # no x_out
    check(got_h, h, th, "h")
    after = pkg.block_norm_params(d, kind=pkg.NORM_LAYER, post=True, pre=False)   # the block's norm alone, nothing to add it to
    r, tr, _, _ = reference(pkg, after, None, y, None, post_w, post_b, None, None)
    out = torch.zeros(6, d, dtype=torch.float16, device="cuda")
    pkg.block_norm(None, y, out, None, 6, after, post_w=post_w, post_b=post_b)
    check(out, r, tr, "x_out")
    plain = pkg.block_norm_params(d, pre=False)                              # an addition
    r, tr, _, _ = reference(pkg, plain, x, y, None, None, None, None, None)
    pkg.block_norm(x, y, out, None, 6, plain)
    check(out, r, tr, "x_out")
    bare = pkg.block_norm_params(d, post=True)                               # norms without weights
    r, tr, h, th = reference(pkg, bare, x, y, None, None, None, None, None)
    got_r, got_h = run(pkg, bare, 6, x, y, None, None, None, None, None)
    check(got_r, r, tr, "x_out")
    check(got_h, h, th, "h")


@pytest.mark.parametrize("d,stride,offset", [(16, 24, 0), (120, 120, 8), (61, 61, 0), (61, 69, 8), (61, 65, 0), (1999, 2007, 0), (200, 208, 0), (400, 400, 0), (700, 704, 8), (4096, 4104, 0), (64, 72, 0), (64, 72, 8), (64, 65, 3), (1000, 1008, 0), (1000, 1001, 1), (1033, 1040, 2)])
def test_strides_and_alignment_and_rows_behind(pkg, torch_cuda, d, stride, offset):
    rows = 11
    def inside(dtype, fill):
        store = torch.full((offset + (rows + 1) * stride,), fill, dtype=dtype, device="cuda")
        return store, store[offset:offset + rows * stride].view(rows, stride)[:, :d]
    x0, y0, g0, *w = inputs(rows, d, torch.float16, torch.float16, True, 3)
    (_, x), (_, y), (_, g), (so, out), (sh, h) = inside(torch.float16, 1.0), inside(torch.float16, 1.0), inside(torch.float16, 1.0), inside(torch.float16, 777.0), inside(torch.float16, 777.0)
    x.copy_(x0), y.copy_(y0), g.copy_(g0)
    bp = pkg.block_norm_params(d, post=True, gate=pkg.GATE_PLAIN, gate_rows=True, x_stride=stride, y_stride=stride, out_stride=stride, h_stride=stride, gate_stride=stride)
    r, tr, hr, th = reference(pkg, bp, x0, y0, g0, *w)
    pkg.block_norm(x, y, out, h, rows - 1, bp, g, *w)
    check(out[:-1], r[:-1], tr[:-1], "x_out")
    check(h[:-1], hr[:-1], th[:-1], "h")
    for store, view in ((so, out), (sh, h)):
        view[:-1] = 777
        assert torch.all(store == 777)                                       # the last row, gaps and ends


def test_rows_that_are_alike_are_equal_whatever_stands_beside_them(pkg, torch_cuda):
    """A row's bits do not depend on the number of rows, nor on its place among them; of an odd width on how it lies to 16 bytes, as which thread adds what does."""
    for d in (48, 200, 512, 1000, 4096, 2049, 333):
        x, y, g, *w = inputs(1, d, torch.float16, torch.float16, False, 4)
        bp = pkg.block_norm_params(d, post=True, gate=pkg.GATE_SIGMOID)
        one = run(pkg, bp, 1, x, y, g, *w)
        many = run(pkg, bp, 6001, x.expand(6001, d).contiguous(), y.expand(6001, d).contiguous(), g, *w)
        for a, b in zip(one, many):
            b = b[::1 if d % 8 == 0 else 8]
            assert torch.equal(a.expand(len(b), d), b)


@pytest.mark.parametrize("d", [96, 4096, 1337])
def test_in_place(pkg, torch_cuda, d):
    x, y, g, *w = inputs(300, d, torch.float16, torch.float16, True, 5)
    bp = pkg.block_norm_params(d, post=True, gate=pkg.GATE_PLAIN, gate_rows=True)
    want = run(pkg, bp, 300, x, y, g, *w)
    pkg.block_norm(x, y, x, y, 300, bp, g, *w)
    assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_what_is_not_finite_stays_in_its_row(pkg, torch_cuda):
    for d in (64, 4096, 1001):
        x, y, g, *w = inputs(8, d, torch.float16, torch.float16, False, 6)
        bp = pkg.block_norm_params(d, post=True, eps=1e-5)
        clean = run(pkg, bp, 8, x, y, None, *w)
        x[1, d // 2], x[3, 0], y[5, d - 1] = float("nan"), float("inf"), float("-inf")
        x_out, h = run(pkg, bp, 8, x, y, None, *w)
        for b in (0, 2, 4, 6, 7):
            assert torch.equal(x_out[b], clean[0][b]) and torch.equal(h[b], clean[1][b])
        assert torch.isnan(x_out[1]).sum() == 1 and torch.isnan(h[1]).all() and torch.isinf(x_out[3]).sum() == 1
        assert torch.isnan(x_out[5]).any() and torch.isnan(h[5]).all()


def test_rows_of_zeros_and_extremes(pkg, torch_cuda):
    d = 4096
    bp = pkg.block_norm_params(d, eps=1e-6)
    x = torch.zeros(4, d, dtype=torch.float16, device="cuda")
    x[1], x[2] = 65504, 2.0 ** -24
    x[3] = torch.arange(d, device="cuda") % 2 * 131008 - 65504
    y = torch.zeros_like(x)
    r, tr, h, th = reference(pkg, bp, x, y, None, None, None, None, None)
    got_r, got_h = run(pkg, bp, 4, x, y, None, None, None, None, None)
    check(got_r, r, tr, "x_out")
    check(got_h, h, th, "h")
    layer = pkg.block_norm_params(d, kind=pkg.NORM_LAYER, eps=1e-6)
    _, got_h = run(pkg, layer, 4, x, y, None, None, None, None, None)
    assert torch.all(got_h[:3] == 0)                                         # rows without a spread


def test_no_rows(pkg, torch_cuda):
    h = torch.full((1, 64), 777.0, dtype=torch.float16, device="cuda")
    pkg.block_norm(h, h, h, h, 0, pkg.block_norm_params(64))
    torch.cuda.synchronize()
    assert torch.all(h == 777)


def test_other_stream_graph_and_host_memory(pkg, torch_cuda):
    d, rows = 1024, 33
    x, y, g, *w = inputs(rows, d, torch.float16, torch.float16, False, 7)
    bp = pkg.block_norm_params(d, post=True, gate=pkg.GATE_SIGMOID)
    want = run(pkg, bp, rows, x, y, g, *w)
    x_out, h = torch.zeros_like(x), torch.zeros_like(x)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            pkg.block_norm(x, y, x_out, h, rows, bp, g, *w, stream=side)
            pkg.block_norm(x_out, None, x_out, h, rows, pkg.block_norm_params(d), pre_w=w[2], stream=side)     # a kernel that reads what the one before it writes
    for _ in range(3):
        x_out.zero_(), h.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x_out, want[0])
    check(h, *reference(pkg, pkg.block_norm_params(d), want[0], None, None, None, None, w[2], None)[2:], "h")
    with pytest.raises(pkg.EfaError, match="memory of the host"):
        pkg.block_norm(x.cpu(), y, x_out, h, rows, bp, g, *w)


# As many rows as make a block look ahead to others', dense and with gaps, at the widths where the kernels of fp32 change, and odd ones.
@pytest.mark.parametrize("d,gap", [(500, 0), (512, 8), (1000, 0), (1017, 3), (2049, 0), (2560, 8), (4096, 0), (5001, 0), (6144, 0), (8192, 8), (8200, 0), (12003, 0), (12296, 0), (16384, 0), (16390, 1),
                                   (20001, 0), (32768, 0)])
@pytest.mark.parametrize("x_bits,y_bits", [(32, 32), (16, 32), (32, 16), (16, 16)])
def test_many_rows_of_every_width(pkg, torch_cuda, d, gap, x_bits, y_bits):
    (xt, xk), (yt, yk) = types(pkg, x_bits), types(pkg, y_bits)
    rows = 2500 if d < 2000 else 900 if d < 9000 else 310
    x0, y0, g0, *w = inputs(rows, d, xt, yt, True, d)
    store = [torch.full(((rows + 1) * (d + gap),), 777.0, dtype=t, device="cuda") for t in (xt, yt, torch.float16, torch.float16)]
    x, y, g, h = (s[:rows * (d + gap)].view(rows, d + gap)[:, :d] for s in store)
    x.copy_(x0), y.copy_(y0), g.copy_(g0)
    s = d + gap if gap else 0
    bp = pkg.block_norm_params(d, kind=d % 2, eps=1e-5, post=d % 3 > 0, gate=pkg.GATE_SIGMOID, gate_rows=True, residual_scale=0.75, block_scale=0.5, x_dtype=xk, y_dtype=yk,
                               x_stride=s, y_stride=s, out_stride=s, h_stride=s, gate_stride=s)
    r, tr, hr, th = reference(pkg, bp, x0, y0, g0, *w)
    pkg.block_norm(x, y, x, h, rows, bp, g, *w)
    check(x, r, tr, "x_out")
    check(h, hr, th, "h")
    assert torch.equal(y, y0) and torch.equal(g, g0)
    for view, whole in ((x, store[0]), (h, store[3])):
        view.fill_(777.0)
        assert torch.all(whole == 777)
