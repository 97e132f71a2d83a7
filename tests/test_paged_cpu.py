"""The paged cache on a machine without a GPU: refusals, sizes, and the sources of its kernels."""
import os
import re

import pytest
import torch

from conftest import ROOT

CSRC = os.path.join(ROOT, "eager-flash-attention_b200", "csrc")
AT = 0x10000000          # an address that nothing is read from


def _cache(pkg, dtype=None, **change):
    f = dict(k=AT, v=AT, k_exp=None, v_exp=None, num_pages=10, page_size=16, H_kv=8, d_h=128, dtype=pkg.F16 if dtype is None else dtype, page_stride=0)
    if f["dtype"] == pkg.E4M3:
        f.update(k_exp=AT, v_exp=AT)
    f.update(change)
    return pkg.PagedCache(*f.values())


def _batch(pkg, **change):
    f = dict(q_start=AT, kv_len=AT, pages=AT, num_seqs=3, max_pages=4, tokens=5, max_q=2, max_kv=64)
    f.update(change)
    return pkg.PagedBatch(*f.values())


def test_legal_arguments_have_no_reason(pkg):
    for dtype in (pkg.F16, pkg.E4M3):
        assert pkg.paged_check(_cache(pkg, dtype), _batch(pkg)) is None
        assert pkg.paged_check(_cache(pkg, dtype), _batch(pkg), pkg.paged_attention_params(32, 128)) is None
    assert pkg.paged_check(_cache(pkg), _batch(pkg, num_seqs=0, tokens=0, max_q=0, max_kv=0)) is None


@pytest.mark.parametrize("change,why", [
    (dict(dtype=0), "EFA_F16 or EFA_E4M3"), (dict(d_h=96), "d_h"), (dict(d_h=256), "d_h"), (dict(page_size=8), "page_size"), (dict(page_size=24), "page_size"),
    (dict(page_size=512), "page_size"), (dict(H_kv=0), "H_kv"), (dict(num_pages=0), "num_pages"), (dict(k=None), "k and v"), (dict(v=AT + 8), "16-byte"),
    (dict(dtype=2, k_exp=None, v_exp=AT), "k_exp"), (dict(dtype=2, k_exp=AT + 4, v_exp=AT), "k_exp"), (dict(page_stride=8 * 16 * 128 - 16), "page_stride"),
    (dict(page_stride=8 * 16 * 128 + 8), "page_stride")])
def test_caches_that_are_refused(pkg, change, why):
    assert why in pkg.paged_check(_cache(pkg, **change), _batch(pkg))
    with pytest.raises(pkg.EfaError, match=why):
        pkg.cache_write(AT, AT, _cache(pkg, **change), _batch(pkg))
    with pytest.raises(pkg.EfaError, match=why):
        pkg.cache_read(AT, AT, _cache(pkg, **change), _batch(pkg))
    with pytest.raises(pkg.EfaError, match=why):
        pkg.paged_attention(AT, AT, _cache(pkg, **change), _batch(pkg), pkg.paged_attention_params(8, 128))


@pytest.mark.parametrize("change,why", [
    (dict(num_seqs=-1), "negative"), (dict(tokens=-1), "negative"), (dict(max_q=-1), "negative"), (dict(max_kv=-1), "negative"), (dict(max_pages=0), "max_pages"),
    (dict(q_start=None), "null"), (dict(kv_len=None), "null"), (dict(pages=None), "null"), (dict(num_seqs=1 << 20, max_pages=1 << 20), "too large"),
    (dict(max_kv=(1 << 30) + 1), "too large"), (dict(max_q=(1 << 30) + 1), "too large"), (dict(tokens=(1 << 30) + 1), "too large")])
def test_batches_that_are_refused(pkg, change, why):
    assert why in pkg.paged_check(_cache(pkg), _batch(pkg, **change))
    with pytest.raises(pkg.EfaError, match=why):
        pkg.cache_write(AT, AT, _cache(pkg), _batch(pkg, **change))


@pytest.mark.parametrize("change,why", [
    (dict(H_q=0), "H_q"), (dict(H_q=12), "H_q"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=0.0), "scale"), (dict(scale=-0.1), "scale"),
    (dict(q_head_stride=640), "strides"), (dict(q_head_stride=640, q_token_stride=132), "strides"), (dict(q_head_stride=64, q_token_stride=128), "strides"),
    (dict(o_token_stride=1016), "o_token_stride"), (dict(o_token_stride=1028), "o_token_stride")])
def test_attention_parameters_that_are_refused(pkg, change, why):
    ap = pkg.paged_attention_params(8, 128)
    for name, value in change.items():
        setattr(ap, name, value)
    assert why in pkg.paged_check(_cache(pkg), _batch(pkg), ap)
    with pytest.raises(pkg.EfaError, match=why):
        pkg.paged_attention_workspace(_cache(pkg), _batch(pkg), ap)
    with pytest.raises(pkg.EfaError, match=why):
        pkg.paged_attention(AT, AT, _cache(pkg), _batch(pkg), ap)


def test_rows_that_are_refused(pkg):
    c, b, ap = _cache(pkg), _batch(pkg), pkg.paged_attention_params(8, 128)
    for call in (pkg.cache_write, pkg.cache_read):
        with pytest.raises(pkg.EfaError, match="null"):
            call(None, AT, c, b)
        with pytest.raises(pkg.EfaError, match="aligned"):
            call(AT, AT + 2, c, b)
        for head, token in ((0, 128), (640, 0), (644, 128), (640, 100), (128, 128), (640, 136), (136, 1024)):
            with pytest.raises(pkg.EfaError, match="strides"):
                call(AT, AT, c, b, head_stride=head, token_stride=token)
    with pytest.raises(pkg.EfaError, match="aligned"):
        pkg.paged_attention(AT + 4, AT, c, b, ap)
    with pytest.raises(pkg.EfaError, match="null"):
        pkg.paged_attention(AT, None, c, b, ap)


def test_a_workspace_that_is_missing_or_short_is_refused(pkg):
    c, b, ap = _cache(pkg), _batch(pkg, max_pages=4096, max_kv=65536), pkg.paged_attention_params(32, 128)
    need = pkg.paged_attention_workspace(c, b, ap)
    assert need > 0
    for at, size in ((None, 0), (AT, need - 1), (AT + 8, need)):
        with pytest.raises(pkg.EfaError, match="workspace"):
            pkg.paged_attention(AT, AT, c, b, ap, at, workspace_bytes=size)
    assert pkg.paged_attention_workspace(c, _batch(pkg), ap) == 0         # 64 keys at most: nothing is cut


def test_empty_batches_launch_nothing(pkg):
    """Without a GPU a launch would fail."""
    ap = pkg.paged_attention_params(8, 128)
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    for b in (_batch(pkg, num_seqs=0), _batch(pkg, tokens=0), _batch(pkg, max_q=0), pkg.paged_batch(i(1), i(0), i(0, 4), 0, 0, 0)):
        for rows in (AT, torch.zeros(8, 0, 128, dtype=torch.float16)):       # an empty tensor has no address
            pkg.cache_write(rows, rows, _cache(pkg), b)
            pkg.cache_read(rows, rows, _cache(pkg), b)
            pkg.paged_attention(rows, rows, _cache(pkg), b, ap)


def test_tensors_that_do_not_fit_together_are_refused(pkg):
    k = torch.zeros(5, 2, 16, 64, dtype=torch.float16)
    e = torch.zeros(5, 2, 16, dtype=torch.uint8)
    c = pkg.paged_cache(k, k.clone())
    assert (c.num_pages, c.H_kv, c.page_size, c.d_h, c.dtype, c.page_stride) == (5, 2, 16, 64, pkg.F16, 2 * 16 * 64)
    both = torch.zeros(5, 2, 2, 16, 64, dtype=torch.float16)               # K and V of a page side by side
    assert pkg.paged_cache(both[:, 0], both[:, 1]).page_stride == 2 * 2 * 16 * 64
    code = k.to(torch.float8_e4m3fn)
    assert pkg.paged_cache(code, code, e, e).dtype == pkg.E4M3 and pkg.paged_cache(code.view(torch.uint8), code.view(torch.uint8), e, e).dtype == pkg.E4M3
    for args in ((k, k[:4]), (k[0], k[0]), (k.float(), k.float()), (k.bfloat16(), k.bfloat16()), (k.transpose(1, 2), k.transpose(1, 2)), (k, k, e, e), (code, code),
                 (code, code, e, None), (code, code, e, e[:4]), (code, code, e, e.int()), (k, code)):
        with pytest.raises(pkg.EfaError):
            pkg.paged_cache(*args)
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    b = pkg.paged_batch(i(4), i(3), i(3, 7), 9, 4, 50)
    assert (b.num_seqs, b.max_pages, b.tokens, b.max_q, b.max_kv) == (3, 7, 9, 4, 50)
    for args in ((i(3), i(3), i(3, 7)), (i(4), i(3), i(2, 7)), (i(4), i(3), i(21)), (i(4).long(), i(3), i(3, 7)), (i(4), i(3), i(7, 3).T)):
        with pytest.raises(pkg.EfaError):
            pkg.paged_batch(*args, 9, 4, 50)


def test_pages_that_overlap_are_refused(pkg):
    one = torch.zeros(1, 2, 16, 64, dtype=torch.float16)
    for pool in (one.expand(5, 2, 16, 64), torch.zeros(2 * 2 * 16 * 64, dtype=torch.float16).as_strided((3, 2, 16, 64), (16 * 64, 16 * 64, 64, 1))):
        with pytest.raises(pkg.EfaError, match="overlap"):
            pkg.paged_cache(pool, pool)
    assert pkg.paged_cache(one, one).page_stride == 0


@pytest.mark.parametrize("at", [0, 1, 2])
@pytest.mark.parametrize("size", [2 ** 31, 2 ** 32, 2 ** 32 + 1, -1])
def test_sizes_of_more_than_31_bits_are_refused(pkg, at, size):
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    sizes = [9, 4, 50]
    sizes[at] = size
    with pytest.raises(pkg.EfaError, match="tokens, max_q and max_kv"):
        pkg.paged_batch(i(4), i(3), i(3, 7), *sizes)


def _kernels():
    """Name and body of every kernel that paged_launch starts."""
    found = {}
    for name in sorted(os.listdir(CSRC)):
        if not name.startswith("paged"):
            continue
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"__global__[^;{]*?\b(paged_\w+_kernel)\(", text):
            depth, i = 0, text.index("{", m.end())
            for at in range(i, len(text)):
                depth += (text[at] == "{") - (text[at] == "}")
                if depth == 0:
                    found[m.group(1)] = text[m.start():at + 1]
                    break
    return found


def test_kernels_that_start_early_presume_no_read_only_memory():
    """They are on the GPU while what they read may still be written (launch_early): a wait ahead of the first access, and ordinary loads."""
    kernels = _kernels()
    assert set(kernels) == {"paged_move_kernel", "paged_rows_kernel", "paged_merge_kernel", "paged_chunk_kernel", "paged_chains_kernel"}
    for name, body in kernels.items():
        assert "pdl_wait()" in body and "pdl_trigger()" in body, name
        assert not re.search(r"__restrict__|__ldg\b|\.nc\b|__constant__", body), name
        assert not re.search(r"paged_seq|paged_part|c\.q_start|c\.kv_len|a\.Q\b|rows\.k", body.split("pdl_wait()", 1)[0].split("{", 1)[-1]), name
