"""How large a batch over the paged cache may be: host arithmetic."""
import pytest

AT = 0x10000000          # an address that nothing is read from


def _why(pkg, seqs, max_q, max_kv, tokens, heads=32, kv_heads=8, page=64, bits=16, d=128):
    e = (None, None) if bits == 16 else (AT, AT)
    cache = pkg.PagedCache(AT, AT, *e, 1000, page, kv_heads, d, pkg.F16 if bits == 16 else pkg.E4M3, 0)
    batch = pkg.PagedBatch(AT, AT, AT, seqs, -(-max_kv // page), tokens, max_q, max_kv)
    return pkg.paged_check(cache, batch, pkg.paged_attention_params(heads, d))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("seqs,max_q,max_kv,tokens", [
    (128, 4096, 131072, 8192), (256, 2048, 131072, 8192), (256, 8192, 32768, 8192),      # chunks among tokens, 8192 rows in all
    (1024, 8192, 1 << 20, 8192), (1024, 4, 1 << 20, 4096), (1, 1 << 18, 1 << 18, 1 << 18)])
def test_batches_of_a_server_are_legal(pkg, bits, seqs, max_q, max_kv, tokens):
    assert _why(pkg, seqs, max_q, max_kv, tokens, bits=bits) is None


@pytest.mark.parametrize("seqs,max_q,max_kv,tokens", [
    (1 << 16, 1 << 20, 4096, 1 << 20),                # items
    (1024, 1 << 20, 1 << 20, 1 << 27),                # units of all items
    (1, (1 << 30) - 1, 4096, 8)])                     # rows of a chunk
def test_what_31_bits_do_not_count_is_refused(pkg, seqs, max_q, max_kv, tokens):
    assert "too large" in _why(pkg, seqs, max_q, max_kv, tokens)
