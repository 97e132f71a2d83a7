"""Shapes of the rows that the norms and the 4-bit projections are given: those of other rows are refused, not read as what they are not."""
import pytest
import torch

AT = 0x10000000


def half(*shape):
    return torch.zeros(*shape, dtype=torch.float16)


def refusal(pkg, call):
    """What the call was refused for; without a GPU it is refused at last, its tensors being the host's."""
    with pytest.raises(pkg.EfaError) as e:
        call()
    return str(e.value)


def w4(pkg, d_in=256, d_out=48):
    return pkg.W4(AT, AT, None, d_in, d_out, 64, 0, 0, 0)


@pytest.mark.parametrize("shape,rows,stride", [
    ((3, 512), 3, 0), ((1, 512), 1, 0), ((6, 128), 2, 0), ((4, 200), 3, 0), ((2, 2, 512), 3, 0), ((5, 3, 128), 3, 0),
    ((3, 200), 2, 200), ((3, 512), 3, 256), ((3, 256), 4, 256), ((5, 3, 256), 2, 768 * 2 - 256), ((3, 5, 256), 6, 512)])
def test_rows_of_another_length_are_refused(pkg, shape, rows, stride):
    X, bp = half(*shape), pkg.block_norm_params(256, x_stride=stride)
    assert "project_w4: X" in refusal(pkg, lambda: pkg.project_w4(X, w4(pkg), half(rows, 48), rows, x_stride=stride))
    assert "block_norm: x" in refusal(pkg, lambda: pkg.block_norm(X, None, None, half(rows, 256), rows, bp))


@pytest.mark.parametrize("shape,rows,stride", [
    ((3, 256), 3, 0), ((3, 256), 2, 0), ((768,), 3, 0), ((800,), 3, 0), ((3, 4, 64), 3, 0), ((2, 3, 256), 6, 0), ((2, 3, 256), 5, 0), ((1, 256), 1, 0), ((256,), 1, 0), ((1, 3, 1, 256), 3, 0),
    ((2, 768), 6, 0), ((12, 64), 3, 0), ((1, 768), 3, 0),
    ((3, 256), 3, 256), ((6, 256), 3, 512), ((5, 256), 3, 512), ((2000,), 3, 512), ((3, 512), 3, 512), ((2, 3, 256), 6, 256), ((1, 512), 1, 300), ((3, 4, 256), 6, 512), ((3, 4, 256), 3, 1024)])
def test_rows_that_are_taken(pkg, shape, rows, stride):
    X, bp = half(*shape), pkg.block_norm_params(256, x_stride=stride)
    stride8 = stride if stride % 8 == 0 else 0
    for why in ([refusal(pkg, lambda: pkg.project_w4(X, w4(pkg), half(rows, 48), rows, x_stride=stride))] if stride8 == stride else []) + \
            [refusal(pkg, lambda: pkg.block_norm(X, None, None, half(rows, 256), rows, bp))]:
        assert "shape" not in why and "dense" not in why and ("memory" in why or "CUDA" in why), why


def test_views_with_their_strides(pkg):
    """Columns of a wider tensor, heads of a wider one, rows of a batch that lie apart by more than a row."""
    whole, w = half(7, 3, 8, 64), w4(pkg, 256)
    for X, rows, stride, taken in ((half(5, 600)[:, 8:264], 5, 600, True), (half(5, 600)[:, 8:], 5, 600, True), (half(5, 600)[:, 8:264], 5, 608, False), (half(5, 600)[1:4, :256], 4, 600, False),
                                   (whole[:, 0, :4], 7, 3 * 512, True), (whole[:, :, :4], 21, 512, True), (whole[:, :2, :4], 14, 512, False), (whole[:, :2, :4], 2, 512, True),
                                   (whole[:, 1, 4:], 7, 512, False), (half(5, 600)[::2, :256], 3, 1200, True)):
        why = refusal(pkg, lambda: pkg.project_w4(X, w, half(rows, 48), rows, x_stride=stride))
        assert ("shape" not in why and "dense" not in why) if taken else ("shape" in why or "beyond" in why), (tuple(X.shape), stride, why)


def test_outputs_and_weights_are_looked_at_too(pkg):
    bp = pkg.block_norm_params(64, post=True, gate=pkg.GATE_PLAIN, gate_rows=True)
    good = dict(x=half(3, 64), y=half(3, 64), x_out=half(3, 64), h=half(3, 64))
    rest = dict(gate=half(3, 64), post_w=half(64), pre_w=half(1, 64))
    assert "shape" not in refusal(pkg, lambda: pkg.block_norm(*good.values(), 3, bp, **rest))
    for name in good:
        bad = {**good, name: half(3, 96)}
        assert f"block_norm: {name}: a tensor of shape [3, 96] is not 3 rows of 64" in refusal(pkg, lambda: pkg.block_norm(*bad.values(), 3, bp, **rest))
    assert "block_norm: gate: a tensor of shape [3, 96]" in refusal(pkg, lambda: pkg.block_norm(*good.values(), 3, bp, **{**rest, "gate": half(3, 96)}))
    assert "block_norm: pre_w: a tensor of shape [1, 96]" in refusal(pkg, lambda: pkg.block_norm(*good.values(), 3, bp, **{**rest, "pre_w": half(1, 96)}))
    assert "project_w4: out: a tensor of shape [3, 96]" in refusal(pkg, lambda: pkg.project_w4(half(3, 256), w4(pkg), half(3, 96), 3))


def test_a_row_of_one_element(pkg):
    bp = pkg.block_norm_params(1)
    assert "shape" in refusal(pkg, lambda: pkg.block_norm(half(4, 2), None, None, half(4, 1), 4, bp))
    assert "shape" not in refusal(pkg, lambda: pkg.block_norm(half(4, 1), None, None, half(4), 4, bp))
    assert "shape" not in refusal(pkg, lambda: pkg.block_norm(half(2, 2), None, None, half(4, 1), 4, bp))


def test_workspaces_that_are_not_dense_are_refused(pkg):
    """An expanded byte has as many elements as one likes, and one byte of memory; what lies between the rows of a view is not the call's."""
    ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32)  # noqa: E731
    pool, cache = pkg.page_pool(ints(10), ints(3, 4), ints(3), 16), pkg.PagedCache(AT, AT, None, None, 10, 16, 8, 128, pkg.F16, 0)
    batch, ap = pkg.paged_batch(ints(4), ints(3), ints(3, 4), 3, 1, 64), pkg.paged_attention_params(16, 128)
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 12, 1 << 9, dtype=torch.uint8)[:, :256]):
        for call in (lambda: pkg.pages_take(pool, ints(4), ws), lambda: pkg.pages_fork(pool, cache, ints(1), ints(1), ws),
                     lambda: pkg.pages_compact(pool, cache, ints(3, 4), ints(10), ints(10), ws), lambda: pkg.paged_attention(AT, AT, cache, batch, ap, ws)):
            assert "the workspace must be a dense tensor" in refusal(pkg, call)
    dense = torch.zeros(1 << 20, dtype=torch.uint8)
    for call in (lambda: pkg.pages_take(pool, ints(4), dense), lambda: pkg.paged_attention(AT, AT, cache, batch, ap, dense)):
        assert "dense" not in refusal(pkg, call)
