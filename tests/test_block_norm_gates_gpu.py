"""A block's norm through gates far from zero: where exp of the gate overflows, where it is a subnormal, and infinite ones.

Tolerance, with u = 2^-24 and e = exp(-|g|): exp is off by 2 + 1.173 |g| units in the last place, twice as many u, of e, and by 2^-149 where e is a subnormal, of
which g < 0 takes the whole and g >= 0 an e of 1 + e; a sum, a reciprocal and two products are 8 u. The residual, the scale and the rounding: 4 u of the magnitudes that are
added, half a step of the type (2^-11 and 2^-25 of fp16, 2^-24 and 2^-149 of fp32)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float("inf")
GATES = [0.0, 0.5, -0.5, 8.0, -8.0, 20.0, -20.0, 60.0, -60.0, 87.25, -87.25, 87.5, -87.5, 88.5, -88.5, 88.75, -88.75, 90.0, -90.0, 100.0, -100.0, 103.0, -103.0, 110.0, -110.0,
         1000.0, -1000.0, 65504.0, -65504.0, INF, -INF]


def gates(rows, d, values=None):
    g = torch.tensor(values or GATES, dtype=torch.float16, device="cuda")
    return g[torch.arange(rows * d, device="cuda") % len(g)].reshape(rows, d)


def exact(y, g):
    e = torch.exp(-g.double().abs())
    return y.double() * torch.where(g < 0, e, torch.ones_like(e)) / (1 + e), e


# Dense rows whose chunks are whole, rows of odd widths with ends, rows that begin anywhere, and rows that are read in their turn.
@pytest.mark.parametrize("d,offset", [(64, 0), (4096, 0), (2049, 0), (333, 0), (500, 1), (32768, 0), (20001, 0)])
@pytest.mark.parametrize("wide", [False, True])
def test_gates_far_from_zero(pkg, torch_cuda, d, offset, wide):
    """The block's output alone, so that nothing hides what is small; fp32 goes up to 2^127."""
    rows, dtype = 5, torch.float32 if wide else torch.float16
    gen = torch.Generator(device="cuda").manual_seed(d)
    y = torch.randn(rows, d, generator=gen, device="cuda")
    y = y.clamp(-1.9, 1.9) * 2.0 ** torch.randint(-20, 127, (rows, d), generator=gen, device="cuda").double() if wide else 1000 * y
    y, g = y.to(dtype), gates(rows, d)
    store = torch.zeros(rows * d + offset, dtype=dtype, device="cuda")
    out = store[offset:].view(rows, d)
    kind = pkg.F32 if wide else pkg.F16
    bp = pkg.block_norm_params(d, pre=False, gate=pkg.GATE_SIGMOID, gate_rows=True, block_scale=0.5, x_dtype=kind, y_dtype=kind)
    pkg.block_norm(None, y, out, None, rows, bp, g)
    torch.cuda.synchronize()
    n, e = exact(y, g)
    n, size = 0.5 * n, 0.5 * y.double().abs()
    s = torch.where(g < 0, e, 1.0)
    of_exp = torch.where(g.isinf() | (e < 2.0 ** -160), torch.zeros_like(e), 2 * U * (2 + 1.173 * g.double().abs()) * e)
    tol = size * (8 * U * s + of_exp + torch.where(g < 0, 2.0 ** -149, 0.0)) + 4 * U * n.abs() + (U * n.abs() + 2.0 ** -149 if wide else 2.0 ** -11 * n.abs() + 2.0 ** -25)
    assert torch.isfinite(out).all()
    worst = ((out.double() - n).abs() / tol).max().item()
    assert worst <= 1, f"{worst:.2f} times the tolerance"
    assert torch.all(out[g == -INF] == 0)


@pytest.mark.parametrize("d", [64, 2049, 32768])
def test_infinite_values_through_gates(pkg, torch_cuda, d):
    """Infinite as long as the gate's exp is a number above zero; through a gate of zero there is no number."""
    rows = 3
    g = gates(rows, d)
    y = torch.full((rows, d), INF, dtype=torch.float16, device="cuda")
    y[:, 1::2] = -INF
    out = torch.zeros_like(y)
    pkg.block_norm(None, y, out, None, rows, pkg.block_norm_params(d, pre=False, gate=pkg.GATE_SIGMOID, gate_rows=True), g)
    torch.cuda.synchronize()
    open_ = g >= -103                                                       # exp(-103) is 2^-148.6
    assert torch.equal(out[open_], y[open_])
    assert torch.isnan(out[g < -105]).all()


def test_a_gate_that_is_no_number(pkg, torch_cuda):
    d = 64
    y, g = torch.ones(2, d, dtype=torch.float16, device="cuda"), torch.zeros(2, d, dtype=torch.float16, device="cuda")
    g[1, 5] = float("nan")
    out = torch.zeros_like(y)
    pkg.block_norm(None, y, out, None, 2, pkg.block_norm_params(d, pre=False, gate=pkg.GATE_SIGMOID, gate_rows=True), g)
    torch.cuda.synchronize()
    assert torch.isnan(out[1, 5]) and torch.isnan(out).sum() == 1 and torch.all(out[0] == 0.5)
