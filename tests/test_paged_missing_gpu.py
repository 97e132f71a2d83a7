"""The paged key/value cache where pages are missing: attention against the definition in 64 bits."""
import pytest
import torch

from paged_helpers import Batch, Pool, attention_ref, fill_random

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(pkg, torch_cuda):
    pkg.kernel_status_reset()
    yield
    torch.cuda.synchronize()
    pkg.kernel_status_reset()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("H,kv,q", [(2, [600, 700], [1, 1]),               # a block, or a cluster, per item
                                    (2, [9000, 4000], [1, 4]),             # equal shares
                                    (2, [600, 700], [40, 33]),             # tiles of 64 rows
                                    (16, [600, 700], [200, 300])])         # tiles of 256 rows
@pytest.mark.parametrize("missing", ["first", "run", "last", "all"])
def test_keys_of_missing_pages_count_as_zeros(pkg, bits, d, H, kv, q, missing):
    page, G = 32, 2
    batch = Batch(pkg, kv, q, page, seed=d)
    pool = Pool(pkg, batch.num_pages, H, page, d, bits, fill=0)
    fill_random(pool, batch, 1)
    held = -(-kv[1] // page)
    gone = {"first": [0], "run": list(range(5)) + list(range(held // 2, held // 2 + 6)), "last": [held - 1], "all": list(range(held))}[missing]
    table = batch.dev[2].clone()
    for i, at in enumerate(gone):
        table[1, at] = (-1, batch.num_pages, 1 << 30)[i % 3]
    broken = pkg.paged_batch(batch.dev[0], batch.dev[1], table, batch.tokens, batch.max_q, batch.max_kv)
    gen = torch.Generator(device="cuda").manual_seed(7)
    Q = (2 * torch.randn(H * G, batch.tokens, d, generator=gen, device="cuda")).half()
    ap = pkg.paged_attention_params(H * G, d)
    ws = torch.empty(max(16, pkg.paged_attention_workspace(pool.cache, broken, ap)), dtype=torch.uint8, device="cuda")
    O = torch.full((batch.tokens, H * G * d), 777.0, dtype=torch.float16, device="cuda")
    pkg.paged_attention(Q, O, pool.cache, broken, ap, ws)
    torch.cuda.synchronize()
    assert pkg.kernel_status()[:2] == (2, 1)
    for b, n in enumerate(q):
        K, V = pool.values(batch, b, "k").clone(), pool.values(batch, b, "v").clone()
        for at in gone if b == 1 else []:
            K[:, at * page:(at + 1) * page] = 0
            V[:, at * page:(at + 1) * page] = 0
        lo = batch.starts[b]
        ref, tol = attention_ref(Q[:, lo:lo + n].double(), K, V, n, kv[b], d ** -0.5, 1)
        got = O[lo:lo + n].reshape(n, H * G, d).transpose(0, 1).double()
        assert bool(torch.isfinite(got).all()), f"sequence {b}"
        assert float(((got - ref).abs() / tol).max()) <= 1, f"sequence {b}"
