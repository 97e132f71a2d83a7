"""What stands around the block and its cache (norms, 4-bit projections, pages), on a machine without a GPU: refusals, sizes, and the sources of its kernels."""
import math
import os
import re

import pytest
import torch

from conftest import ROOT

CSRC = os.path.join(ROOT, "eager-flash-attention_b200", "csrc")
AT = 0x10000000          # an address that nothing is read from


# ---- norms ---------------------------------------------------------------------------------------------------------------------------------
def test_norm_sizes_that_are_legal(pkg):
    for d in (1, 7, 4096, 32768):
        for kind in (pkg.NORM_RMS, pkg.NORM_LAYER):
            assert pkg.block_norm_check(pkg.block_norm_params(d, kind=kind), 3) is None
    assert pkg.block_norm_check(pkg.block_norm_params(8, x_dtype=pkg.F32, y_dtype=pkg.F32, x_stride=8, eps=0.0), 0) is None


@pytest.mark.parametrize("change,why", [
    (dict(d=0), "d must"), (dict(d=32769), "d must"), (dict(kind=2), "kind"), (dict(kind=-1), "kind"), (dict(gate=3), "gate"), (dict(x_dtype=2), "EFA_F16 or EFA_F32"),
    (dict(y_dtype=-1), "EFA_F16 or EFA_F32"), (dict(eps=-1e-6), "eps"), (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"), (dict(residual_scale=math.inf), "scales"),
    (dict(block_scale=math.nan), "scales"), (dict(x_stride=63), "strides"), (dict(y_stride=-64), "strides"), (dict(out_stride=1), "strides"), (dict(h_stride=63), "strides"),
    (dict(gate_stride=63), "strides")])
def test_norms_that_are_refused(pkg, change, why):
    bp = pkg.block_norm_params(64)
    for name, value in change.items():
        setattr(bp, name, value)
    assert why in pkg.block_norm_check(bp, 1)
    with pytest.raises(pkg.EfaError, match=why):
        pkg.block_norm(AT, AT, AT, AT, 1, bp)


def test_norm_arguments_that_are_refused(pkg):
    bp = pkg.block_norm_params(64)
    assert "negative" in pkg.block_norm_check(bp, -1)
    for args, kw, why in (((None, None, AT, AT), {}, "x and y are null"), ((AT, AT, None, None), {}, "x_out and h are null"), ((AT, AT, AT, AT), dict(gate=AT), "gate")):
        with pytest.raises(pkg.EfaError, match=why):
            pkg.block_norm(*args, 1, bp, **kw)
    with pytest.raises(pkg.EfaError, match="gate"):
        pkg.block_norm(AT, AT, AT, AT, 1, pkg.block_norm_params(64, gate=pkg.GATE_SIGMOID))
    with pytest.raises(pkg.EfaError, match="needs y"):
        pkg.block_norm(AT, None, AT, AT, 1, pkg.block_norm_params(64, post=True))
    with pytest.raises(pkg.EfaError, match="needs y"):
        pkg.block_norm(AT, None, AT, AT, 1, pkg.block_norm_params(64, gate=pkg.GATE_PLAIN), gate=AT)
    with pytest.raises(pkg.EfaError, match="pre norm"):
        pkg.block_norm(AT, AT, AT, AT, 1, pkg.block_norm_params(64, pre=False))
    for at in range(4):
        with pytest.raises(pkg.EfaError, match="aligned"):
            pkg.block_norm(*[AT + (i == at) for i in range(4)], 1, bp)
    with pytest.raises(pkg.EfaError, match="aligned"):
        pkg.block_norm(AT + 2, AT, AT, AT, 1, pkg.block_norm_params(64, x_dtype=pkg.F32))
    pkg.block_norm(AT, AT, AT, AT, 0, bp)                                   # no rows: nothing is looked at


def test_norm_tensors_that_are_refused(pkg):
    half, wide = torch.zeros(3, 64, dtype=torch.float16), torch.zeros(3, 64)
    bp = pkg.block_norm_params(64)
    for args, kw, why in (((wide, half, half, half), {}, "block_norm: x must be torch.float16"), ((half, wide, half, half), {}, "block_norm: y must be torch.float16"),
                          ((half, half, wide, half), {}, "block_norm: x_out"), ((half, half, half, wide), {}, "block_norm: h"), ((half.bfloat16(), half, half, half), {}, "block_norm: x"),
                          ((half, half, half, half), dict(pre_w=torch.zeros(63, dtype=torch.float16)), "block_norm: pre_w must be a dense tensor of 64"),
                          ((half, half, half, half), dict(post_b=torch.zeros(64)), "block_norm: post_b"), ((half[:, :60], half, half, half), {}, "block_norm: x must be a dense"),
                          ((half, half[::2], half, half), {}, "block_norm: y must be a dense")):
        with pytest.raises(pkg.EfaError, match=why):
            pkg.block_norm(*args, 3, bp, **kw)
    with pytest.raises(pkg.EfaError, match="block_norm: x must be a dense tensor of 256"):
        pkg.block_norm(half, half, half, half, 4, bp)
    strided = pkg.block_norm_params(64, x_stride=128)
    with pytest.raises(pkg.EfaError, match="beyond its memory"):
        pkg.block_norm(half, half, half, half, 3, strided)
    with pytest.raises(pkg.EfaError, match="neighbours"):
        pkg.block_norm(torch.zeros(64, 200, dtype=torch.float16).t()[:, :64], half, half, half, 3, strided)


# ---- projections ---------------------------------------------------------------------------------------------------------------------------
def _w4(pkg, **change):
    f = dict(codes=AT, scales=AT, zeros=None, d_in=256, d_out=48, group=64, code_stride=0, scale_stride=0, zero_stride=0)
    f.update(change)
    return pkg.W4(*f.values())


@pytest.mark.parametrize("change,why", [
    (dict(group=16), "group"), (dict(group=256), "group"), (dict(group=0), "group"), (dict(d_in=0), "d_in"), (dict(d_in=-64), "d_in"), (dict(d_in=96), "d_in"), (dict(d_out=0), "d_out"),
    (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(codes=AT + 8), "16-byte"), (dict(scales=AT + 1), "aligned"), (dict(code_stride=112), "code_stride"),
    (dict(code_stride=136), "code_stride"), (dict(scale_stride=47), "scale_stride"), (dict(zero_stride=-1), "zero_stride"), (dict(d_in=(1 << 24) + 64), "too large"),
    (dict(d_out=(1 << 24) + 1), "too large")])
def test_weights_that_are_refused(pkg, change, why):
    with pytest.raises(pkg.EfaError, match=why):
        pkg.project_w4(AT, _w4(pkg, **change), AT, 1)


def test_projections_that_are_refused(pkg):
    w = _w4(pkg)
    for args, kw, why in (((AT, w, AT, -1), {}, "rows"), ((AT, w, AT, (1 << 19) + 1), {}, "rows"), ((AT, w, AT, 1), dict(out_dtype=2), "EFA_F16 or EFA_F32"),
                          ((AT, w, AT, 1), dict(x_stride=248), "x_stride"), ((AT, w, AT, 1), dict(x_stride=260), "x_stride"), ((AT, w, AT, 1), dict(out_stride=47), "out_stride"),
                          ((None, w, AT, 1), {}, "null"), ((AT, w, None, 1), {}, "null"), ((AT + 8, w, AT, 1), {}, "aligned"), ((AT, w, AT + 1, 1), {}, "aligned"),
                          ((AT, w, AT + 2, 1), dict(out_dtype=0), "aligned")):
        with pytest.raises(pkg.EfaError, match=why):
            pkg.project_w4(*args, **kw)
    pkg.project_w4(None, w, None, 0)                                        # no rows: nothing is looked at
    half = torch.zeros(3, 256, dtype=torch.float16)
    for X, out, why in ((half.float(), half, "project_w4: X must be torch.float16"), (half[:2], half, "project_w4: X must be a dense tensor of 768"),
                        (half, half.reshape(-1)[:140], "project_w4: out must be a dense tensor of 144"), (half, half.int(), "project_w4: out")):
        with pytest.raises(pkg.EfaError, match=why):
            pkg.project_w4(X, w, out, 3)


def test_weight_tensors(pkg):
    codes, scales, zeros = torch.zeros(48, 128, dtype=torch.uint8), torch.zeros(4, 48, dtype=torch.float16), torch.zeros(4, 48, dtype=torch.uint8)
    w = pkg.w4_weight(codes, scales, zeros)
    assert (w.d_in, w.d_out, w.group, w.code_stride, w.scale_stride, w.zero_stride) == (256, 48, 64, 128, 48, 48)
    w = pkg.w4_weight(codes[:, :64], scales[:2])                            # a rank's rows: strides of the whole
    assert (w.d_in, w.d_out, w.group, w.code_stride, w.scale_stride, w.zeros) == (128, 48, 64, 128, 48, None)
    w = pkg.w4_weight(codes[16:32], scales[:, 16:32], zeros[:, 16:32])      # a rank's columns
    assert (w.d_in, w.d_out, w.code_stride, w.scale_stride, w.zero_stride) == (256, 16, 128, 48, 48)
    for bad in ((codes.int(), scales), (codes, scales.float()), (codes, scales[:, :47]), (codes, scales[:3]), (codes, scales, zeros.int()), (codes, scales, zeros[:2]),
                (codes.t().contiguous().t(), scales), (codes[:1].expand(48, 128), scales), (codes, scales[:1])):
        with pytest.raises(pkg.EfaError, match="w4"):
            pkg.w4_weight(*bad)


# ---- pages ---------------------------------------------------------------------------------------------------------------------------------
def _pool(pkg, **change):
    f = dict(refs=AT, pages=AT, kv_len=AT, num_pages=10, page_size=16, num_seqs=3, max_pages=4)
    f.update(change)
    return pkg.PagePool(*f.values())


def _cache(pkg, **change):
    f = dict(k=AT, v=AT, k_exp=None, v_exp=None, num_pages=10, page_size=16, H_kv=8, d_h=128, dtype=pkg.F16, page_stride=0)
    f.update(change)
    return pkg.PagedCache(*f.values())


def _calls(pkg, pool, cache, ws=AT, size=1 << 20):
    return [lambda: pkg.pages_take(pool, AT, ws, workspace_bytes=size), lambda: pkg.pages_fork(pool, cache, AT, AT, ws, n=1, workspace_bytes=size),
            lambda: pkg.pages_compact(pool, cache, AT, AT, AT, ws, workspace_bytes=size), lambda: pkg.pages_free(pool, AT, n=1)]


@pytest.mark.parametrize("change,why", [
    (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"), (dict(num_pages=0), "positive"), (dict(max_pages=0), "positive"), (dict(num_seqs=-1), "negative"),
    (dict(refs=None), "refs"), (dict(pages=None), "pages and kv_len"), (dict(kv_len=None), "pages and kv_len"), (dict(num_pages=(1 << 30) + 1), "too large"), (dict(refs=AT + 2), "aligned"), (dict(pages=AT + 1), "aligned"), (dict(kv_len=AT + 3), "aligned"),
    (dict(num_seqs=1 << 20, max_pages=1 << 20), "too large")])
def test_pools_that_are_refused(pkg, change, why):
    pool = _pool(pkg, **change)
    assert pkg.pages_workspace(pool) == 0
    for call in _calls(pkg, pool, _cache(pkg)):
        with pytest.raises(pkg.EfaError, match=why):
            call()


def test_page_calls_that_are_refused(pkg):
    pool, cache = _pool(pkg), _cache(pkg)
    need = pkg.pages_workspace(pool)
    assert need > 0
    for ws, size in ((None, 0), (AT, need - 1), (AT + 8, need)):
        for call in _calls(pkg, pool, cache, ws, size)[:3]:
            with pytest.raises(pkg.EfaError, match="workspace"):
                call()
    for bad, why in ((dict(num_pages=9), "same number"), (dict(page_size=32), "same number"), (dict(d_h=96), "d_h"), (dict(k=None), "k and v")):
        for call in _calls(pkg, pool, _cache(pkg, **bad))[1:3]:
            with pytest.raises(pkg.EfaError, match=why):
                call()
    for n in (-1, 4):
        with pytest.raises(pkg.EfaError, match="slots"):
            pkg.pages_fork(pool, cache, AT, AT, AT, n=n, workspace_bytes=need)
    for n in (-1, 11):
        with pytest.raises(pkg.EfaError, match="number of pages"):
            pkg.pages_copy(cache, AT, AT, n=n)
    with pytest.raises(pkg.EfaError, match="n must"):
        pkg.pages_free(pool, AT, n=-1)
    for call in (lambda: pkg.pages_take(pool, None, AT, workspace_bytes=need), lambda: pkg.pages_fork(pool, cache, None, AT, AT, n=1, workspace_bytes=need),
                 lambda: pkg.pages_free(pool, None, n=1), lambda: pkg.pages_copy(cache, AT, None, n=1), lambda: pkg.pages_compact(pool, cache, AT, None, AT, AT, workspace_bytes=need)):
        with pytest.raises(pkg.EfaError, match="null"):
            call()
    for call in (lambda: pkg.pages_take(pool, AT + 2, AT, workspace_bytes=need), lambda: pkg.pages_fork(pool, cache, AT, AT + 1, AT, n=1, workspace_bytes=need),
                 lambda: pkg.pages_free(pool, AT + 2, n=1), lambda: pkg.pages_copy(cache, AT + 1, AT, n=1), lambda: pkg.pages_compact(pool, cache, AT, AT, AT + 2, AT, workspace_bytes=need)):
        with pytest.raises(pkg.EfaError, match="aligned"):
            call()
    pkg.pages_fork(pool, cache, None, None, AT, n=0, workspace_bytes=need)                  # nothing to do: nothing is looked at
    pkg.pages_free(pool, None, n=0)
    pkg.pages_copy(cache, None, None, n=0)
    pkg.pages_take(_pool(pkg, num_seqs=0), None, None, workspace_bytes=0)


def test_page_tensors_that_are_refused(pkg):
    i = lambda *shape: torch.zeros(*shape, dtype=torch.int32)  # noqa: E731
    for bad in ((i(10).long(), i(3, 4), i(3)), (i(10), i(3, 4).t(), i(4)), (i(10), i(3, 4), i(4)), (i(10, 1), i(3, 4), i(3)), (i(10), i(12), i(3))):
        with pytest.raises(pkg.EfaError, match="page_pool"):
            pkg.page_pool(*bad, 16)
    with pytest.raises(pkg.EfaError, match="page_size"):
        pkg.page_pool(i(10), i(3, 4), i(3), 24)
    pool = pkg.page_pool(i(10), i(3, 4), i(3), 16)
    assert (pool.num_pages, pool.page_size, pool.num_seqs, pool.max_pages) == (10, 16, 3, 4)
    with pytest.raises(pkg.EfaError, match="q_start must be a dense int32 tensor of 4"):
        pkg.pages_take(pool, i(3), AT, workspace_bytes=1 << 20)
    with pytest.raises(pkg.EfaError, match="seqs must be"):
        pkg.pages_free(pool, i(3).long())
    with pytest.raises(pkg.EfaError, match="src and dst must be as many"):
        pkg.pages_copy(_cache(pkg), i(2), i(1))
    with pytest.raises(pkg.EfaError, match="children must be a dense int32 tensor of 2"):
        pkg.pages_fork(pool, _cache(pkg), i(2), i(1), AT, n=2, workspace_bytes=1 << 20)
    with pytest.raises(pkg.EfaError, match="parents and children must be as many"):
        pkg.pages_fork(pool, _cache(pkg), i(2), i(1), AT, workspace_bytes=1 << 20)
    with pytest.raises(pkg.EfaError, match="moved must be"):
        pkg.pages_compact(pool, _cache(pkg), i(3, 4), i(10), i(9), AT, workspace_bytes=1 << 20)


# ---- sources -------------------------------------------------------------------------------------------------------------------------------
def test_kernels_wait_before_they_read(pkg):
    """They are launched while the kernel ahead of them may still run."""
    for name, kernels in (("block_norm.cu", 1), ("proj_w4_sm100.cu", 1), ("proj_w4_tc_sm100.cu", 1), ("pages.cu", 5)):
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        bodies = text.split("__global__")[1:]
        assert len(bodies) >= kernels
        for body in bodies:
            assert "pdl_wait();" in body and "pdl_trigger();" in body
        assert not re.search(r"__restrict__|__ldg\b|global\.nc\b|__constant__", text)
