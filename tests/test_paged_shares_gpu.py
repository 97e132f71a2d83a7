"""The launch of a full batch of single tokens: large shares for most blocks, small ones for those that start last."""
import pytest
import torch

from paged_helpers import Batch, Pool, check_attention, fill_random

pytestmark = pytest.mark.gpu

LATE_UNITS, LATE_RATIO = 4, 10                            # paged_args.cuh
UNIT, EXTRA, TILE, PER_SM = 64, 1, 16, 2                  # paged_kernels.cuh, fp16 heads of 64 and 128


def _blocks(pkg, pool, batch, ap):
    """Blocks of equal shares, from the workspace: 32 bytes and two places of TILE rows (O and two numbers) each."""
    each = 2 * TILE * (pool.d + 2) * 4
    size = pkg.paged_attention_workspace(pool.cache, batch.batch, ap)
    return next((n for n in range(1, 2000) if (n * 32 + 255) // 256 * 256 + n * each == size), 0)


@pytest.mark.parametrize("d,H,kv", [(64, 8, [9001 - 60 * i for i in range(16)]), (128, 8, [9000] * 12), (128, 3, [36000 + i for i in range(8)] + [1, 0, 700])])
@pytest.mark.parametrize("G,q", [(1, 1), (4, 3)])
def test_unequal_shares(pkg, torch_cuda, d, H, kv, G, q):
    pkg.kernel_status_reset()
    batch = Batch(pkg, kv, [q] * len(kv), 64, seed=d)
    pool = Pool(pkg, batch.num_pages, H, 64, d, 16)
    fill_random(pool, batch, 1)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    big, late = sms * PER_SM, sms * PER_SM * 3 // 4
    ap = pkg.paged_attention_params(H * G, d)
    assert _blocks(pkg, pool, batch, ap) == big + late                       # planned, ...
    weight = H * sum(max(1, -(-n // UNIT)) + EXTRA for n in kv)
    assert weight // LATE_UNITS >= big * LATE_RATIO + late                   # ... and taken with these lengths
    Q = 2 * torch.randn(H * G, batch.tokens, d, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    Q = Q.half()
    ws = torch.full((pkg.paged_attention_workspace(pool.cache, batch.batch, ap),), 0xFF, dtype=torch.uint8, device="cuda")
    outs = []
    for _ in range(2):
        O = torch.full((batch.tokens, H * G * d), 777.0, dtype=torch.float16, device="cuda")
        pkg.paged_attention(Q, O, pool.cache, batch.batch, ap, ws)
        torch.cuda.synchronize()
        check_attention(O, Q, pool, batch, d ** -0.5, 1)
        outs.append(O)
    assert torch.equal(*outs) and pkg.kernel_status()[0] == 0


def test_lengths_that_shrink_under_the_same_plan(pkg, torch_cuda):
    """Unequal shares are planned by the bounds; with shorter sequences the blocks find equal ones, or none."""
    kv = [9000] * 16
    batch = Batch(pkg, kv, [1] * 16, 64)
    pool = Pool(pkg, batch.num_pages, 8, 64, 64, 16)
    fill_random(pool, batch, 1)
    Q = torch.randn(32, 16, 64, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").half()
    ap = pkg.paged_attention_params(32, 64)
    ws = torch.empty(pkg.paged_attention_workspace(pool.cache, batch.batch, ap), dtype=torch.uint8, device="cuda")
    for lengths in ([9000] * 16, [9000] + [1] * 15, [700] * 16, [5 * i for i in range(16)]):
        batch.kv = list(lengths)
        batch.dev[1].copy_(torch.tensor(lengths, dtype=torch.int32))
        O = torch.full((16, 32 * 64), 777.0, dtype=torch.float16, device="cuda")
        pkg.paged_attention(Q, O, pool.cache, batch.batch, ap, ws)
        torch.cuda.synchronize()
        check_attention(O, Q, pool, batch, 0.125, 1)
