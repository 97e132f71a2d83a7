"""Attention over the paged cache where value rows differ in size: every element against the definition in 64 bits."""
import pytest
import torch

from paged_helpers import Batch, Pool, check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("H,kv,q", [(2, [900, 61], [1, 4]), (2, [9000, 4000], [1, 4]), (2, [600, 700], [40, 33]), (16, [600, 700], [200, 300])])
@pytest.mark.parametrize("large", ["one", "some", "small"])
def test_value_rows_of_unlike_size(pkg, bits, d, H, kv, q, large):
    """Values of one token, or of some, that are 2^8 to 2^22 times the others', in a few columns; in the rest the others are all there is."""
    batch = Batch(pkg, kv, q, 32, seed=d)
    pool = Pool(pkg, batch.num_pages, H, 32, d, bits)
    gen = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    for b, n in enumerate(kv):
        V = 0.003 * rnd(H, n, d)
        at = {"one": [0], "some": list(range(0, n, 37)), "small": list(range(n - 1))}[large]
        V[:, at] = 0
        for i, key in enumerate(at):
            V[:, key, i % 3] = 2.0 ** (i % 15) * 3.4
        pool.put(batch, b, "v", V.half())
        pool.put(batch, b, "k", rnd(H, n, d).half())
    Q = rnd(2 * H, batch.tokens, d).half()
    ap = pkg.paged_attention_params(2 * H, d)
    ws = torch.empty(max(16, pkg.paged_attention_workspace(pool.cache, batch.batch, ap)), dtype=torch.uint8, device="cuda")
    O = torch.empty(batch.tokens, 2 * H * d, dtype=torch.float16, device="cuda")
    pkg.paged_attention(Q, O, pool.cache, batch.batch, ap, ws)
    torch.cuda.synchronize()
    check_attention(O, Q, pool, batch, d ** -0.5, 1)
