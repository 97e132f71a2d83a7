"""A paged cache in plain form: batches, pools and the definitions in 64 bits, for the tests of the paged operators."""
import math
import random

import torch

NAN_CODE = 0x7F


def grid():
    """The 127 magnitudes of e4m3, by their bits."""
    return torch.tensor([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (x - 7) for x in range(1, 16) for m in range(8) if (x, m) != (15, 7)],
                        dtype=torch.float64)


def decode(code, byte):
    """Values of codes (uint8 [..., d]) with exponent bytes [...]."""
    table = torch.cat([grid(), torch.tensor([math.nan], dtype=torch.float64)]).to(code.device)
    table = torch.cat([table, -table])
    return table[code.long()] * torch.exp2(byte.double() - 127)[..., None]


def encode(x):
    """(codes, exponent bytes) of rows x, from the definition: nearest grid point of x / 2^e, ties to the even code."""
    x = x.double()
    good = torch.isfinite(x)
    top = torch.where(good, x.abs(), torch.zeros_like(x)).amax(-1)
    e = torch.full_like(top, -24.0)
    for power in range(-24, 8):
        e = torch.where(top > 448 * 2.0 ** power, torch.full_like(e, power + 1.0), e)
    g = grid().to(x.device)
    y = torch.where(good, x.abs(), torch.zeros_like(x)) / torch.exp2(e)[..., None]
    up = torch.searchsorted(g, y.contiguous()).clamp(max=len(g) - 1)
    down = (up - 1).clamp(min=0)
    a, b = g[up] - y, y - g[down]
    code = torch.where((b < a) | ((b == a) & (down % 2 == 0)), down, up)
    code = torch.where(e[..., None] == 8, code.clamp(max=int((g == 240).nonzero()[0, 0])), code)
    code = code + 128 * torch.signbit(x).long()
    code = torch.where(good, code, torch.full_like(code, NAN_CODE))
    return code.to(torch.uint8), (e + 127).to(torch.uint8)


class Batch:
    """Sequences with kv[b] keys, of which the last q[b] are the chunk, on pages in random order."""

    def __init__(self, pkg, kv, q, page, seed=0, spare=3, extra_rows=0, max_q=None, max_kv=None, width=None, first_row=0):
        rng = random.Random(seed)
        self.pkg, self.kv, self.q, self.page = pkg, list(kv), list(q), page
        held = [-(-n // page) for n in self.kv]
        self.num_pages = sum(held) + spare
        order = list(range(self.num_pages))
        rng.shuffle(order)
        self.width = width or max(1, max(held, default=1))
        self.table = [[0] * self.width for _ in self.kv]
        at = 0
        for b, n in enumerate(held):
            self.table[b][:n] = order[at:at + n]
            at += n
        self.starts = [first_row]
        for n in self.q:
            self.starts.append(self.starts[-1] + n)
        self.tokens = self.starts[-1] + extra_rows
        self.max_q = max(self.q, default=0) if max_q is None else max_q
        self.max_kv = max(self.kv, default=0) if max_kv is None else max_kv
        self.dev = [torch.tensor(x, dtype=torch.int32).cuda() for x in (self.starts, self.kv, self.table)]
        self.dev[2] = self.dev[2].reshape(len(self.kv), self.width)
        self.batch = pkg.paged_batch(*self.dev, self.tokens, self.max_q, self.max_kv)

    def places(self, b, lo, hi):
        """Pages and slots of keys [lo, hi) of sequence b."""
        at = torch.arange(lo, hi)
        return torch.tensor(self.table[b])[at // self.page], at % self.page


class Pool:
    """k and v (and exponents) of a cache on the GPU, filled with `fill` bytes."""

    def __init__(self, pkg, num_pages, H, page, d, bits, fill=0xFF, gap=0):
        self.bits, self.H, self.d, self.page = bits, H, d, page
        n = H * page * d
        def one():
            store = torch.full((num_pages, (n + gap) * (2 if bits == 16 else 1)), fill, dtype=torch.uint8, device="cuda")
            store = store.view(torch.float16) if bits == 16 else store
            return store.as_strided((num_pages, H, page, d), (n + gap, page * d, d, 1))
        self.k, self.v = one(), one()
        self.k_exp = self.v_exp = None
        if bits == 8:
            self.k_exp, self.v_exp = (torch.full((num_pages, H, page), fill, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.cache = pkg.paged_cache(self.k, self.v, self.k_exp, self.v_exp)

    def values(self, batch, b, name):
        """fp64 [H][kv][d] of sequence b."""
        page, slot = batch.places(b, 0, batch.kv[b])
        x = getattr(self, name)[page.cuda(), :, slot.cuda()]
        if self.bits == 8:
            return decode(x, getattr(self, name + "_exp")[page.cuda(), :, slot.cuda()]).transpose(0, 1)
        return x.double().transpose(0, 1)

    def put(self, batch, b, name, rows):
        """Values [H][kv][d] (fp16) of sequence b, written by torch."""
        page, slot = (x.cuda() for x in batch.places(b, 0, batch.kv[b]))
        if self.bits == 8:
            code, byte = encode(rows)
            getattr(self, name)[page, :, slot] = code.transpose(0, 1)
            getattr(self, name + "_exp")[page, :, slot] = byte.transpose(0, 1)
        else:
            getattr(self, name)[page, :, slot] = rows.half().transpose(0, 1)


def fill_random(pool, batch, seed, spread=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for b, n in enumerate(batch.kv):
        for name in ("k", "v"):
            pool.put(batch, b, name, spread * torch.randn(pool.H, n, pool.d, generator=gen, device="cuda"))


def attention_ref(q, K, V, n, kv, scale, causal):
    """(O, tolerance), both fp64 [H_q][n][d], of one sequence: q [H_q][n][d], K and V [H_kv][kv][d] in fp64.

    Rows that see nothing are zero; a key that a row does not see has no part in it, whatever its value is.

    Tolerance, with w the weights, A = sum w |v|, u = 2^-11 (half a step of fp16): the weights are rounded to fp16 for the product with V, u A, or 2^-25 a
    weight below 2^-14: 2^-25 sum |v| / l; the result is rounded, u |O| or 2^-25. Scores are sums of d products in fp32, off by (d + 4) 2^-23 sum |q k| scale
    at most (the tensor cores may cut instead of round), ex2 by 2^-22 and its argument's rounding by |s| 2^-22: twice their sum relative to
    A, once above and once below the line. Sums over the keys in fp32: kv 2^-23 A."""
    H_q, G, d = q.shape[0], q.shape[0] // K.shape[0], K.shape[2]
    K, V = K.repeat_interleave(G, 0), V.repeat_interleave(G, 0)
    last = torch.arange(kv - n, kv, device=q.device) if causal else torch.full((n,), kv - 1, device=q.device)
    sees = torch.arange(kv, device=q.device)[None] <= last[:, None]
    s = (q @ K.transpose(1, 2)) * scale
    size = (q.abs() @ K.abs().transpose(1, 2)) * scale
    s = torch.where(sees, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True) if kv else torch.zeros(H_q, n, 1, dtype=torch.float64, device=q.device)
    p = torch.where(sees, torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top)), torch.zeros_like(s))
    l = p.sum(-1, keepdim=True)
    bad = ~torch.isfinite(V)
    clean = torch.where(bad, torch.zeros_like(V), V)
    none = ~sees.any(-1)[None, :, None]
    div = torch.where(none, torch.ones_like(l), l)
    O = p @ clean / div
    if bad.any():                                   # whatever is not finite and seen makes the element so
        O = torch.where(sees.double() @ bad.double() > 0, torch.full_like(O, math.nan), O)
    O = torch.where(none, torch.zeros_like(O), O)
    A = p @ clean.abs() / div
    big = torch.where(sees, size, torch.zeros_like(size)).amax(-1, keepdim=True) if kv else l
    off = 2 * ((d + 4) * 2.0 ** -23 * big + 2.0 ** -22 * (1 + 1.45 * big)) + kv * 2.0 ** -23
    tol = 2.0 ** -11 * (A + O.nan_to_num().abs()) + 2.0 ** -25 * (1 + (sees.double() @ clean.abs()) / div) + A * off
    return O, tol * 1.01


def check_attention(O, q, pool, batch, scale, causal, skip=()):
    """O [tokens][H_q * d] against the reference, sequence by sequence; returns the worst error over its tolerance."""
    H_q, d, worst = q.shape[0], q.shape[2], 0.0
    for b, n in enumerate(batch.q):
        if n == 0 or b in skip:
            continue
        lo = batch.starts[b]
        ref, tol = attention_ref(q[:, lo:lo + n].double(), pool.values(batch, b, "k"), pool.values(batch, b, "v"), n, batch.kv[b], scale, causal)
        got = O[lo:lo + n].reshape(n, H_q, d).transpose(0, 1).double()
        assert torch.equal(torch.isfinite(got), torch.isfinite(ref)), f"sequence {b}: other elements are finite"
        err = ((got - ref).abs() / tol).nan_to_num()
        worst = max(worst, float(err.max()))
        assert worst <= 1, f"sequence {b}: {worst:.2f} times the tolerance at {err.argmax().item()}"
    return worst
