"""What writing to the paged cache and reading it back report of lengths that are wrong."""
import pytest
import torch

from paged_helpers import Batch, Pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
def test_write_and_read_report_wrong_lengths_of_any_sequence(pkg, torch_cuda, bits):
    n = 300
    batch = Batch(pkg, [50] * n, [0 if b % 3 == 1 else 1 for b in range(n)], 16)
    pool = Pool(pkg, batch.num_pages, 3, 16, 64, bits)
    K = torch.randn(3, batch.tokens, 64, device="cuda").half()
    V = torch.randn(3, batch.tokens, 64, device="cuda").half()
    calls = (lambda: pkg.cache_write(K, V, pool.cache, batch.batch), lambda: pkg.cache_read(torch.empty_like(K), torch.empty_like(V), pool.cache, batch.batch))
    for which, index, value, seqs in ((1, 1, 51, (1,)), (1, 298, -1, (298,)), (1, 299, 1 << 30, (299,)), (0, n, 5, (n - 1,)), (0, 0, -3, (0,)), (0, 100, 0, (99, 100)),
                                      (0, n, batch.tokens + 1, (n - 1,))):
        x = batch.dev[which]
        good = x[index].item()
        for call in calls:
            pkg.kernel_status_reset()
            x[index] = value
            call()
            torch.cuda.synchronize()
            code, seq, site, _ = pkg.kernel_status()
            assert (code, site) == (3, 50) and seq in seqs, (which, index, value)
            x[index] = good
            pkg.kernel_status_reset()
            call()
            torch.cuda.synchronize()
            assert pkg.kernel_status()[0] == 0
