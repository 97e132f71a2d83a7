"""Batches over the paged cache with bounds far above their lengths, at the most that a legal batch may have, and beyond."""
import random

import pytest
import torch

from paged_helpers import Batch, Pool, check_attention, fill_random

pytestmark = pytest.mark.gpu


def _attend(pkg, q, pool, batch, causal=1):
    ap = pkg.paged_attention_params(q.shape[0], q.shape[2], causal)
    O = torch.full((q.shape[1], q.shape[0] * q.shape[2]), 777.0, dtype=torch.float16, device="cuda")
    ws = torch.full((max(16, pkg.paged_attention_workspace(pool.cache, batch, ap)),), 0xFF, dtype=torch.uint8, device="cuda")
    pkg.paged_attention(q, O, pool.cache, batch, ap, ws)
    torch.cuda.synchronize()
    return O


def _rows(*shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").half()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("seqs,max_q,max_kv", [(128, 4096, 131072), (256, 2048, 131072), (256, 8192, 32768)])
def test_a_chunk_among_many_tokens_with_loose_bounds(pkg, torch_cuda, bits, seqs, max_q, max_kv):
    pkg.kernel_status_reset()
    rng = random.Random(seqs)
    kv = [rng.randint(1, 200) for _ in range(seqs)]
    q = [1] * seqs
    kv[5], q[5] = 900, 300
    batch = Batch(pkg, kv, q, 64, max_q=max_q, max_kv=max_kv, width=max_kv // 64, extra_rows=8192 - sum(q))
    pool = Pool(pkg, batch.num_pages, 8, 64, 128, bits)
    fill_random(pool, batch, 1)
    Q = _rows(32, batch.tokens, 128)
    O = _attend(pkg, Q, pool, batch.batch)
    check_attention(O, Q, pool, batch, 128 ** -0.5, 1)
    assert torch.all(O[batch.starts[-1]:] == 777) and pkg.kernel_status()[0] == 0


@pytest.mark.parametrize("bits", [16, 8])
def test_a_batch_of_all_the_work_that_is_legal(pkg, torch_cuda, bits):
    """Chunks that just begin another tile, every sequence as long as the bound, no mask."""
    pkg.kernel_status_reset()
    batch = Batch(pkg, [9088] * 4, [65] * 4, 64)
    pool = Pool(pkg, batch.num_pages, 8, 64, 64, bits)
    fill_random(pool, batch, 1)
    Q = _rows(32, batch.tokens, 64)
    check_attention(_attend(pkg, Q, pool, batch.batch, 0), Q, pool, batch, 0.125, 0)
    assert pkg.kernel_status()[0] == 0


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("d", [64, 128])
def test_sequences_with_rows_in_common_are_reported(pkg, torch_cuda, bits, d):
    """... and where they add up to more than any legal batch has, in equal shares, nothing is computed."""
    pkg.kernel_status_reset()
    one = Batch(pkg, [9000], [512], 64)
    pool = Pool(pkg, one.num_pages, 8, 64, d, bits)
    fill_random(pool, one, 1)
    Q = _rows(32, 512, d)
    n = 40
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = pkg.paged_batch(i32(*[512 * (b % 2) for b in range(n + 1)]), i32(*[9000] * n), one.dev[2].expand(n, -1).contiguous(), 512, 512, 9000)
    O = _attend(pkg, Q, pool, batch)
    assert pkg.kernel_status()[0] == 3 and torch.all(O == 777)
    pkg.kernel_status_reset()
    check_attention(_attend(pkg, Q, pool, one.batch), Q, pool, one, d ** -0.5, 1)      # the next call is as ever
    assert pkg.kernel_status()[0] == 0
