"""Scores far from zero over the paged cache: products of fp16 rows that are finite give results that are, from every kernel."""
import math

import pytest
import torch

from paged_helpers import Batch, Pool, check_attention

pytestmark = pytest.mark.gpu

KERNELS = [(2, 2, 128, [900], [1]), (2, 1, 64, [20000], [1]), (2, 2, 128, [700], [40]), (8, 4, 128, [900, 300], [300, 40]), (16, 2, 64, [1500], [1000]), (8, 4, 128, [6000], [70]),
           (16, 1, 16, [4000], [700]), (8, 2, 32, [3000], [260])]


def _attend(pkg, Q, pool, batch, scale):
    ap = pkg.paged_attention_params(Q.shape[0], Q.shape[2], 1, scale)
    ws = torch.empty(max(16, pkg.paged_attention_workspace(pool.cache, batch.batch, ap)), dtype=torch.uint8, device="cuda")
    O = torch.empty(Q.shape[1], Q.shape[0] * Q.shape[2], dtype=torch.float16, device="cuda")
    pkg.paged_attention(Q, O, pool.cache, batch.batch, ap, ws)
    torch.cuda.synchronize()
    return O


def _pool(pkg, batch, H, d, bits, keys):
    """keys: of sequence b, [kv][d]; values at random."""
    pool = Pool(pkg, batch.num_pages, H, 64, d, bits)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for b, n in enumerate(batch.kv):
        pool.put(batch, b, "k", keys(b, n).half().cuda().expand(H, n, d))
        pool.put(batch, b, "v", torch.randn(H, n, d, generator=gen, device="cuda").half())
    return pool


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("H,G,d,kv,q", KERNELS)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
def test_the_largest_score_takes_all(pkg, torch_cuda, bits, H, G, d, kv, q, sign, order):
    """Scores of up to 2^34, exact in fp32, 10^7 and more apart or equal: a row is the mean of the values of its largest."""
    batch = Batch(pkg, kv, q, 64)

    def keys(b, n):
        j = torch.arange(n)
        level = {"rising": j, "falling": n - 1 - j, "mixed": j * 7919 % 1009}[order] * 15 // max(n, 1009) + 8       # 8 to 22: exact in four bits where even or below 16
        level = torch.where(level > 15, level // 2 * 2, level)
        return (level * 2048.0)[:, None].expand(n, d)

    pool = _pool(pkg, batch, H, d, bits, keys)
    Q = torch.full((H * G, batch.tokens, d), sign * 16384.0, dtype=torch.float16, device="cuda")
    O = _attend(pkg, Q, pool, batch, d ** -0.5)
    for b, n in enumerate(q):
        V, level = pool.values(batch, b, "v"), pool.values(batch, b, "k")[0, :, 0] * sign
        top = torch.cummax(level, 0).values
        for i in range(0, n, 7):
            last = kv[b] - n + i
            best = level[:last + 1] == top[last]
            want = V[:, :last + 1][:, best].mean(1)                                      # [H][d]
            got = O[batch.starts[b] + i].reshape(H, G, d).double()
            # weights of 1 and fp32 sums, then fp16: 2^-11 of the values' size, and as much again for the sums
            assert float((got - want[:, None]).abs().max()) <= 2.0 ** -10 * float(V.abs().max())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("H,G,d,kv,q", KERNELS)
@pytest.mark.parametrize("centre", [1000, 4096, 30000])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_near_one_another_far_from_zero(pkg, torch_cuda, bits, H, G, d, kv, q, centre, sign):
    """Powers of 2 to the `centre`, give or take 6."""
    batch = Batch(pkg, kv, q, 64)

    def keys(b, n):
        j = torch.arange(n)
        x = torch.zeros(n, d)
        x[:, 0] = 2048
        x[:, 1] = (j * 31 % 13 - 6) * 64 + j * 17 % 64                                    # of 2048 / 32: 1 in the power
        return x

    pool = _pool(pkg, batch, H, d, bits, keys)
    Q = torch.zeros(H * G, batch.tokens, d, dtype=torch.float16, device="cuda")
    Q[:, :, 0], Q[:, :, 1] = sign * centre / 32, 1
    check_attention(_attend(pkg, Q, pool, batch, math.log(2) / 64), Q, pool, batch, math.log(2) / 64, 1)
