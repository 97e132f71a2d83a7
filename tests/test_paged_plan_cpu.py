"""Which launch attention over the paged cache takes, told by its workspace: a block per item needs none."""
import pytest

AT = 0x10000000          # an address that nothing is read from


def _workspace(pkg, seqs, tokens, max_q, max_kv, heads, kv_heads, d, bits):
    e = (None, None) if bits == 16 else (AT, AT)
    cache = pkg.PagedCache(AT, AT, *e, 10000, 64, kv_heads, d, pkg.F16 if bits == 16 else pkg.E4M3, 0)
    batch = pkg.PagedBatch(AT, AT, AT, seqs, -(-max_kv // 64), tokens, max_q, max_kv)
    return pkg.paged_attention_workspace(cache, batch, pkg.paged_attention_params(heads, d))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("heads,kv_heads,d", [(32, 8, 128), (16, 16, 64), (32, 32, 128)])
@pytest.mark.parametrize("chunk,others,max_kv", [(4096, 127, 4096), (512, 63, 4096), (4096, 255, 4096)])
def test_a_chunk_among_single_tokens_goes_in_shares(pkg, bits, heads, kv_heads, d, chunk, others, max_kv):
    """Not as a block for each tile that every sequence might have."""
    assert _workspace(pkg, others + 1, chunk + others, chunk, max_kv, heads, kv_heads, d, bits) > 0


@pytest.mark.parametrize("heads,kv_heads,d", [(32, 8, 128), (16, 16, 64)])
def test_prompts_go_by_item(pkg, heads, kv_heads, d):
    assert _workspace(pkg, 1, 4096, 4096, 4096, heads, kv_heads, d, 16) == 0
    assert _workspace(pkg, 8, 8 * 2048, 2048, 2048, heads, kv_heads, d, 16) == 0
