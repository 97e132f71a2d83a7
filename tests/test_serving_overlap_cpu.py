"""Outputs that lie in what a call reads: in place where the header says so, in the gaps of strided rows, refused otherwise. Host arithmetic on addresses."""
import pytest

AT = 0x10000000          # an address that nothing is read from


def refusal(pkg, call):
    with pytest.raises(pkg.EfaError) as e:
        call()
    return str(e.value)


def norm(pkg, rows, d, x, y, x_out, h, gate=None, gate_rows=False, pre_w=None, **kw):
    bp = pkg.block_norm_params(d, gate=pkg.GATE_PLAIN if gate else pkg.GATE_NONE, gate_rows=gate_rows, **kw)
    return refusal(pkg, lambda: pkg.block_norm(x, y, x_out, h, rows, bp, gate, pre_w=pre_w))


B = 0x20000000           # far from AT, so is C
C = 0x30000000


def test_norms_in_place(pkg):
    for args in ((AT, B, AT, B), (AT, B, B, AT), (AT, B, C, AT), (AT, B, None, B), (AT, None, AT, B)):
        assert "overlap" not in norm(pkg, 9, 64, *args)
    assert "overlap" not in norm(pkg, 9, 64, AT, B, AT, C, x_dtype=pkg.F32)
    assert "overlap" not in norm(pkg, 9, 64, AT, B, AT, B, x_stride=96, out_stride=96, y_stride=72, h_stride=72)
    assert "overlap" not in norm(pkg, 1, 64, AT, B, AT, B, x_stride=96)     # one row has no stride


def test_norms_that_would_lose_what_they_read(pkg):
    assert "x_out overlaps y" in norm(pkg, 9, 64, AT, B, B, C, x_dtype=pkg.F32)                       # another type
    assert "h overlaps x" in norm(pkg, 1, 64, AT, B, C, AT, x_dtype=pkg.F32)
    assert "h overlaps y" in norm(pkg, 9, 64, AT, B, C, B, y_dtype=pkg.F32)
    assert "x_out overlaps x" in norm(pkg, 9, 64, AT, B, AT, C, x_stride=96)                         # another stride
    assert "x_out overlaps x" in norm(pkg, 9, 64, AT, B, AT + 128, C)                                # a row further on
    assert "h overlaps y" in norm(pkg, 9, 64, AT, B, AT, B + 16)                                     # not whole elements of the same row
    assert "x_out overlaps gate" in norm(pkg, 9, 64, AT, B, C, None, gate=C + 128)                   # one gate for all rows, within the output
    assert "h overlaps pre_w" in norm(pkg, 9, 64, AT, B, AT, C, pre_w=C + 256)
    assert "x_out and h overlap" in norm(pkg, 9, 64, AT, B, C, C + 128)
    assert "x_out and h overlap" in norm(pkg, 9, 64, AT, B, C, C, x_dtype=pkg.F32)


def test_norms_between_rows(pkg):
    """Columns of one tensor: rows of one stride that do not meet."""
    assert "overlap" not in norm(pkg, 9, 64, AT, AT + 128, AT + 256, AT + 384, x_stride=256, y_stride=256, out_stride=256, h_stride=256)
    assert "x_out overlaps y" in norm(pkg, 9, 64, AT, AT + 160, AT + 256, AT + 384, x_stride=256, y_stride=256, out_stride=256, h_stride=256)
    assert "h overlaps x" in norm(pkg, 9, 64, AT, B, AT + 128, AT + 400, x_stride=256, out_stride=256, h_stride=256)     # the last columns and the next row's first


def test_projections(pkg):
    w = pkg.W4(C, C, None, 256, 48, 64, 0, 0, 0)
    call = lambda X, out, rows, **kw: refusal(pkg, lambda: pkg.project_w4(X, w, out, rows, **kw))  # noqa: E731
    assert "overlap" not in call(AT, B, 9)
    assert "overlap" not in call(AT, AT + 9 * 512, 9)
    for out in (AT, AT + 16, AT + 9 * 512 - 2, AT - 2):
        assert "out overlaps X" in call(AT, out, 9), hex(out)
    assert "overlap" not in call(AT, AT + 512, 9, x_stride=304, out_stride=304)                     # columns of one tensor
    assert "out overlaps X" in call(AT, AT + 512, 9, x_stride=304, out_stride=304, out_dtype=pkg.F32)
    assert "out overlaps X" in call(AT, AT + 510, 9, x_stride=304, out_stride=304)


def test_one_row_between_others(pkg):
    """A vector in the gaps of strided rows, and one output row in the gaps of what is read."""
    kw = dict(out_stride=128, h_stride=128)
    assert "overlap" not in norm(pkg, 9, 64, AT, B, C, None, gate=C + 128, **kw)
    assert "x_out overlaps gate" in norm(pkg, 9, 64, AT, B, C, None, gate=C + 64, **kw)
    assert "x_out overlaps gate" in norm(pkg, 9, 64, AT, B, C, None, gate=C + 192, **kw)
    assert "overlap" not in norm(pkg, 9, 64, AT, B, C, C + 128, pre_w=C + 9 * 256, **kw)
    assert "h overlaps pre_w" in norm(pkg, 9, 64, AT, B, C, C + 128, pre_w=C + 128 + 256, **kw)
    assert "x_out and h overlap" in norm(pkg, 1, 64, AT, B, C, C + 64)
    assert "overlap" not in norm(pkg, 1, 64, AT, B, C, C + 128)
