"""Tensors that rows are read from and written to, ahead of the calls on the paged cache."""
import pytest
import torch

AT = 0x10000000          # an address that nothing is read from
H, T, D = 4, 6, 64


def _calls(pkg, K, V, Q, O, heads=8, **strides):
    cache = pkg.PagedCache(AT, AT, None, None, 10, 16, H, D, pkg.F16, 0)
    batch = pkg.PagedBatch(AT, AT, AT, 3, 4, T, 2, 64)
    kv = {k: v for k, v in strides.items() if k in ("head_stride", "token_stride")}
    ap = pkg.paged_attention_params(heads, D, **{k: v for k, v in strides.items() if k not in kv})
    if K is not None:
        pkg.cache_write(K, V, cache, batch, **kv)
        pkg.cache_read(K, V, cache, batch, **kv)
    if Q is not None:
        pkg.paged_attention(Q, O, cache, batch, ap)


def _half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def _reaches_the_library(pkg, *args, **strides):
    """Without a GPU that is where the call ends."""
    with pytest.raises(pkg.EfaError) as e:
        _calls(pkg, *args, **strides)
    assert "rows must be" not in str(e.value) and "beyond its memory" not in str(e.value)


@pytest.mark.skipif(torch.cuda.is_available(), reason="host tensors would reach the checks of memory")
def test_tensors_that_fit_reach_the_library(pkg):
    kv, q, o = _half(H, T, D), _half(8, T, D), _half(T, 8 * D)
    _reaches_the_library(pkg, kv, kv, None, None)
    _reaches_the_library(pkg, None, None, q, o)
    _reaches_the_library(pkg, _half(H * T * D + 5), _half(H, T, D), None, None)
    by_token = _half(T, H, D + 8)
    _reaches_the_library(pkg, by_token, by_token, None, None, head_stride=D + 8, token_stride=H * (D + 8))
    packed = _half(T, 3, H, D)                          # Q, K and V of a token side by side
    _reaches_the_library(pkg, packed[:, 1], packed[:, 2], None, None, head_stride=D, token_stride=3 * H * D)
    long = _half(H, 100, D)
    _reaches_the_library(pkg, long[:, :T], long[:, :T], None, None, head_stride=100 * D, token_stride=D)
    _reaches_the_library(pkg, None, None, q, _half(T, 8 * D + 16)[:, :8 * D], o_token_stride=8 * D + 16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.int16, torch.float8_e4m3fn])
def test_other_types_are_refused(pkg, dtype):
    kv, q, o = _half(H, T, D), _half(8, T, D), _half(T, 8 * D)
    for args in ((kv.to(dtype), kv, None, None), (kv, kv.to(dtype), None, None), (None, None, q.to(dtype), o), (None, None, q, o.to(dtype))):
        with pytest.raises(pkg.EfaError, match="float16"):
            _calls(pkg, *args)


def test_views_without_their_strides_are_refused(pkg):
    kv, q, o = _half(H, T, D), _half(8, T, D), _half(T, 8 * D)
    turned = _half(T, H, D).transpose(0, 1)
    for args in ((turned, kv, None, None), (kv, turned, None, None), (None, None, _half(T, 8, D).transpose(0, 1), o), (None, None, q, _half(8 * D, T).T)):
        with pytest.raises(pkg.EfaError, match="dense"):
            _calls(pkg, *args)


def test_tensors_that_are_too_small_are_refused(pkg):
    kv, q, o = _half(H, T, D), _half(8, T, D), _half(T, 8 * D)
    for args in ((_half(H, T - 1, D), kv, None, None), (kv, _half(H, T, D // 2), None, None), (None, None, _half(7, T, D), o), (None, None, q, _half(T - 1, 8 * D))):
        with pytest.raises(pkg.EfaError, match="dense"):
            _calls(pkg, *args)
    by_token = _half(T, H, D + 8)
    for args, strides in (((by_token[1:], by_token, None, None), dict(head_stride=D + 8, token_stride=H * (D + 8))),
                          ((by_token, by_token, None, None), dict(head_stride=D + 8, token_stride=H * (D + 8) + 16)),
                          ((None, None, _half(T, 8, D), o), dict(q_head_stride=D, q_token_stride=8 * D + 8)), ((None, None, q, o), dict(o_token_stride=8 * D + 8))):
        with pytest.raises(pkg.EfaError, match="beyond its memory"):
            _calls(pkg, *args, **strides)
