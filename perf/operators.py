"""The operators of the paged key/value cache, case by case: writing rows of keys and values into pages (fp16, or e4m3 with an exponent per
row), reading them back, and attention of a chunk of new tokens over the pages. `run` computes them as elementary torch operations, or, where
`own` is true, through the package.

A batch is ragged: sequence b has kv_len[b] keys in the cache, of which the last q_len[b] are the chunk's; their rows are packed one
sequence after another. Row i of the chunk stands at position kv_len - q_len + i and sees the keys up to there.
"""
import importlib
import math

import torch

own = False

EXP_MIN, EXP_BIAS = -24, 127


# ---- cases ---------------------------------------------------------------------------------------------------------------------------------
# op        what one pass does: "write" (rows into pages of fp16), "keep" (rows into pages and back out of them), "read" (pages into rows), "attend"
# seqs      sequences of the batch; q, q_min, kv, kv_min: most and fewest rows and keys of a sequence
# heads     query heads (attend only); kv_heads; d_h; page: keys to a page; bits: 16 (fp16) or 8 (e4m3)
def _case(name, op, seqs, q, q_min, kv, kv_min, heads, kv_heads, d_h, page, bits):
    return dict(name=name, op=op, seqs=seqs, q=q, q_min=q_min, kv=kv, kv_min=kv_min, heads=heads, kv_heads=kv_heads, d_h=d_h, page=page, bits=bits)


def listed():
    return [
        # one user's next token, after its projection: a call of a few kilobytes
        _case("write_one_token", "write", 1, 1, 1, 1000, 1000, 16, 16, 64, 64, 16),
        # a prompt of several users, chunk by chunk, every head with keys of its own
        _case("write_prompts", "write", 4, 2048, 901, 8192, 2048, 32, 32, 128, 64, 16),
        # the next tokens of a full batch into a cache of 8 bits, and back for a check or a copy elsewhere
        _case("keep_tokens_8bit", "keep", 64, 1, 1, 4096, 1, 32, 8, 128, 16, 8),
        # prompts into a cache of 8 bits, and back as the attention over contiguous keys wants them
        _case("keep_prompts_8bit", "keep", 6, 4096, 333, 8192, 4096, 32, 8, 128, 32, 8),
        # whole sequences out of the pages: handing them to another process, or to the attention over contiguous keys
        _case("read_sequences", "read", 8, 16384, 517, 16384, 517, 16, 16, 64, 16, 16),
        _case("read_sequences_8bit", "read", 5, 32768, 4099, 32768, 4099, 32, 8, 128, 128, 8),
        # one user's next token: latency
        _case("token_one_user", "attend", 1, 1, 1, 1000, 1000, 16, 16, 64, 64, 16),
        # the next tokens of a full batch, heads in groups
        _case("tokens_batch", "attend", 64, 1, 1, 8192, 129, 32, 8, 128, 64, 16),
        # long contexts in 8 bits, a few tokens each as in speculative decoding
        _case("tokens_long_8bit", "attend", 16, 4, 1, 32768, 2051, 32, 8, 128, 32, 8),
        # a prompt from its first token on, every head with keys of its own
        _case("prompt_fresh", "attend", 1, 4096, 4096, 4096, 4096, 16, 16, 64, 64, 16),
        # a chunk of a long document
        _case("chunk_long", "attend", 1, 2048, 2048, 32768, 32768, 32, 8, 128, 128, 16),
        # prompts in chunks and single tokens in one batch, 8 bits
        _case("chunks_mixed_8bit", "attend", 12, 512, 1, 8192, 640, 32, 8, 128, 16, 8),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "keep", "read", "attend", "attend", "attend"])
    d_h = rng.choice([16, 32, 64, 64, 128, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
    heads = kv_heads * rng.choice([g for g in (1, 1, 2, 3, 4, 7, 8) if kv_heads * g <= 64])
    page, bits = rng.choice([16, 32, 64, 128, 256]), 16 if op == "write" else rng.choice([16, 8])
    while True:
        seqs = _log_int(rng, 1, 128)
        kv = _log_int(rng, 1, 32768)
        kv_min = _log_int(rng, 1, kv)
        if op == "read":
            q, q_min = kv, kv_min
        else:
            q = 1 if rng.random() < 0.3 else _log_int(rng, 1, min(kv, 4096))
            q_min = rng.choice([1, q, _log_int(rng, 1, q)])
        c = dict(op=op, seqs=seqs, q=q, q_min=q_min, kv=kv, kv_min=kv_min, heads=heads, kv_heads=kv_heads, d_h=d_h, page=page, bits=bits)
        cells = seqs * heads * q * kv if op == "attend" else 0             # scores of the plain form
        if cells <= 1 << 30 and seqs * (kv + page) * kv_heads * d_h <= 1 << 28:
            return c


def _spread(b, most, fewest):
    """Sequence 0 has the most, the others something in between, each its own. (Of rows, every third sequence has the fewest.)"""
    return most if b == 0 else fewest + (most - fewest) * ((b * 40503 + 9973) % 65536) // 65535


def _lengths(case):
    kv = [_spread(b, case["kv"], case["kv_min"]) for b in range(case["seqs"])]
    if case["op"] == "read":
        return kv, kv
    return kv, [min(n, case["q_min"] if b % 3 == 1 else _spread(b * 7, case["q"], case["q_min"])) for b, n in enumerate(kv)]


def work(case):
    kv, q = _lengths(case)
    row = case["kv_heads"] * case["d_h"]                                   # elements of one token's keys
    kept = 2 * row * (case["bits"] // 8) + (2 * case["kv_heads"] if case["bits"] == 8 else 0)       # bytes of one token in the cache
    tokens = sum(q)
    if case["op"] != "attend":
        return {"bytes": tokens * (4 * row + kept) * (2 if case["op"] == "keep" else 1), "flops": 0}
    seen = sum(n * (2 * k - n + 1) // 2 for k, n in zip(kv, q))            # (row, key) pairs of a head
    return {"bytes": sum(kv) * kept + tokens * case["heads"] * case["d_h"] * 4, "flops": 4 * case["d_h"] * case["heads"] * seen}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------------
def _quantised(x):
    """Codes (fp32 values on the e4m3 grid) and exponents of rows x: x ~ code * 2^exponent."""
    top = x.abs().amax(-1, keepdim=True)
    fraction, exponent = torch.frexp(top)                                   # top = fraction * 2^exponent, fraction in [1/2, 1)
    e = torch.where(fraction > 0.875, exponent - 8, exponent - 9).clamp(min=EXP_MIN)       # 448 = 0.875 * 2^9
    e = torch.where(top > 0, e, torch.full_like(e, EXP_MIN))
    code = torch.ldexp(x, -e)
    step = torch.ldexp(torch.ones_like(x), torch.frexp(code).exponent.clamp(min=-5) - 4)   # three bits behind the first; 2^-9 at the bottom
    most = torch.where(e == 8, 240.0, 448.0)                                # 256 * 2^8 is no fp16
    return ((code / step).round() * step).clamp(-most, most), e             # round() takes ties to even


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    kv, q = _lengths(case)
    H, d, page = case["kv_heads"], case["d_h"], case["page"]
    per_seq = -(-case["kv"] // page)
    need = sum(-(-n // page) for n in kv)
    pool = need + 3
    order = torch.randperm(pool, generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    table = torch.zeros(case["seqs"], per_seq, dtype=torch.int32)
    place, at = torch.full((case["seqs"], per_seq), -1, dtype=torch.int64), 0
    for b, n in enumerate(kv):
        held = -(-n // page)
        place[b, :held] = torch.arange(at, at + held)
        at += held
    place = place.cuda()
    table = torch.where(place >= 0, order[place.clamp(min=0)], torch.zeros_like(table.cuda())).to(torch.int32)
    starts = [0]
    for n in q:
        starts.append(starts[-1] + n)
    s = {"case": case, "q_start": torch.tensor(starts, dtype=torch.int32).cuda(), "kv_len": torch.tensor(kv, dtype=torch.int32).cuda(),
         "pages": table, "tokens": starts[-1]}

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    shape = (pool, H, page, d)
    for name in ("k", "v"):
        if case["op"] in ("write", "keep"):
            s[name] = torch.zeros(shape, dtype=torch.float16 if case["bits"] == 16 else torch.uint8, device="cuda")
            if case["bits"] == 8:
                s[name + "_exp"] = torch.zeros(shape[:3], dtype=torch.uint8, device="cuda")
        elif case["bits"] == 16:
            s[name] = normal(*shape).half()
        else:
            code, e = _quantised(normal(*shape).half().float())
            s[name] = code.to(torch.float8_e4m3fn).view(torch.uint8)
            s[name + "_exp"] = (e.squeeze(-1) + EXP_BIAS).to(torch.uint8)
    if case["op"] in ("write", "keep"):
        s["K"], s["V"] = normal(H, s["tokens"], d).half(), normal(H, s["tokens"], d).half()
    if case["op"] == "attend":
        s["Q"] = (2 * normal(case["heads"], s["tokens"], d)).half()
        s["O"] = torch.zeros(s["tokens"], case["heads"] * d, dtype=torch.float16, device="cuda")
    elif case["op"] != "write":
        s["K_out"], s["V_out"] = (torch.zeros(H, s["tokens"], d, dtype=torch.float16, device="cuda") for _ in range(2))
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------------------
def _slots(s):
    """Page and place in it of every row of the chunk."""
    token = torch.arange(s["tokens"], device="cuda", dtype=torch.int64)
    seq = torch.searchsorted(s["q_start"][1:].long(), token, right=True)
    position = s["kv_len"].long()[seq] - s["q_start"].long()[seq + 1] + token
    return s["pages"].long()[seq, position // s["case"]["page"]], position % s["case"]["page"]


def _stored(s, name):
    """The values of a whole pool, in fp32."""
    if s["case"]["bits"] == 16:
        return s[name].float()
    return torch.ldexp(s[name].view(torch.float8_e4m3fn).float(), s[name + "_exp"].to(torch.int32).unsqueeze(-1) - EXP_BIAS)


def _put(s, name, rows):
    page, place = _slots(s)
    if s["case"]["bits"] == 16:
        s[name][page, :, place] = rows.transpose(0, 1)
        return
    code, e = _quantised(rows.float())
    s[name][page, :, place] = code.to(torch.float8_e4m3fn).view(torch.uint8).transpose(0, 1)
    s[name + "_exp"][page, :, place] = (e.squeeze(-1) + EXP_BIAS).to(torch.uint8).transpose(0, 1)


def _get(s, name):
    page, place = _slots(s)
    rows = s[name][page, :, place]
    if s["case"]["bits"] == 16:
        return rows.transpose(0, 1).contiguous()
    e = s[name + "_exp"][page, :, place].to(torch.int32).unsqueeze(-1) - EXP_BIAS
    return torch.ldexp(rows.view(torch.float8_e4m3fn).float(), e).half().transpose(0, 1).contiguous()


def _attend(s):
    c = s["case"]
    B, H, G, d, n = c["seqs"], c["kv_heads"], c["heads"] // c["kv_heads"], c["d_h"], c["q"]
    keys = s["pages"].shape[1] * c["page"]
    index = s["pages"].long()
    K, V = (_stored(s, x)[index].permute(0, 2, 1, 3, 4).reshape(B, H, 1, keys, d) for x in ("k", "v"))
    i = torch.arange(n, device="cuda")
    start, length = s["q_start"].long()[:-1, None], (s["q_start"][1:] - s["q_start"][:-1]).long()[:, None]
    there = i < length                                                      # [B, n]: a row of this sequence
    row = torch.where(there, start + i, torch.full_like(start + i, s["tokens"]))
    Q = torch.cat([s["Q"].float(), torch.zeros(c["heads"], 1, d, device="cuda")], 1)[:, row].reshape(H, G, B, n, d).permute(2, 0, 1, 3, 4)
    last = s["kv_len"].long()[:, None] - length + i                         # the last key that a row sees
    sees = (torch.arange(keys, device="cuda") <= last[..., None])[:, None, None]
    score = (Q @ K.transpose(-1, -2)).mul_(1 / math.sqrt(d)).masked_fill_(~sees, -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    O = (p @ V) / p.sum(-1, keepdim=True)
    out = torch.zeros(s["tokens"] + 1, c["heads"] * d, dtype=torch.float16, device="cuda")
    out[row] = O.permute(0, 3, 1, 2, 4).reshape(B, n, H * G * d).half()
    return out[:-1]


# ---- through the package -------------------------------------------------------------------------------------------------------------------
class _Call:
    """What a program keeps for the calls on one cache and one batch."""

    def __init__(self, s):
        c, self.pkg = s["case"], importlib.import_module("eager-flash-attention_b200")
        self.device = s["k"].device.index
        self.cache = self.pkg.paged_cache(s["k"], s["v"], s.get("k_exp"), s.get("v_exp"))
        self.batch = self.pkg.paged_batch(s["q_start"], s["kv_len"], s["pages"], s["tokens"], c["q"], c["kv"])
        if c["op"] == "attend":
            self.how = self.pkg.paged_attention_params(c["heads"], c["d_h"], causal=1)
            size = self.pkg.paged_attention_workspace(self.cache, self.batch, self.how)
            self.workspace = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None


def _through_package(s):
    call = s.get("call")
    if call is None:
        call = s["call"] = _Call(s)
    pkg, op, stream = call.pkg, s["case"]["op"], torch._C._cuda_getCurrentRawStream(call.device)    # the current stream, without 3 us for an object of it
    if op == "attend":
        pkg.paged_attention(s["Q"], s["O"], call.cache, call.batch, call.how, call.workspace, stream=stream)
        return s["O"]
    if op != "read":
        pkg.cache_write(s["K"], s["V"], call.cache, call.batch, stream=stream)
        if op == "write":
            return {"k": s["k"], "v": s["v"]}
    pkg.cache_read(s["K_out"], s["V_out"], call.cache, call.batch, stream=stream)
    return {"K": s["K_out"], "V": s["V_out"]}


def run(state):
    if own:
        return _through_package(state)
    op = state["case"]["op"]
    if op == "attend":
        return _attend(state)
    if op != "read":
        _put(state, "k", state["K"])
        _put(state, "v", state["V"])
        if op == "write":
            return {"k": state["k"], "v": state["v"]}
    return {"K": _get(state, "k"), "V": _get(state, "v")}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------------
def _grid():
    """All e4m3 magnitudes, the smallest first: m/8 * 2^-6, then (1 + m/8) * 2^(x - 7)."""
    at = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** (x - 7) for x in range(1, 16) for m in range(8)]
    return torch.tensor(at[:-1], dtype=torch.float64, device="cuda")       # the last pattern is NaN


def _value_kept(x):
    """What a row of 64-bit numbers is once it went through the cache of 8 bits: the nearest grid point, ties to the even pattern."""
    grid = _grid()
    e = torch.full(x.shape[:-1] + (1,), float(EXP_MIN), dtype=torch.float64, device="cuda")
    top = x.abs().amax(-1, keepdim=True)
    for power in range(EXP_MIN, 8):
        e = torch.where(top > 448 * 2.0 ** power, torch.full_like(e, power + 1.0), e)
    scale = torch.exp2(e)
    y = x.abs() / scale
    above = torch.searchsorted(grid, y.contiguous()).clamp(max=len(grid) - 1)
    below = (above - 1).clamp(min=0)
    to_above, to_below = grid[above] - y, y - grid[below]
    at = torch.where((to_below < to_above) | ((to_below == to_above) & (below % 2 == 0)), below, above)
    return torch.copysign(torch.minimum(grid[at], torch.where(e == 8, 240.0, 448.0).double()) * scale, x)


def exact(case, seed):
    kv, q = _lengths(case)
    if case["op"] == "attend" and sum(k * n for k, n in zip(kv, q)) * case["heads"] * case["d_h"] > 2e13:
        return None
    s = prepare(case, seed)
    page, H, d = case["page"], case["kv_heads"], case["d_h"]
    bits8 = case["bits"] == 8
    table, starts = s["pages"].cpu().tolist(), s["q_start"].cpu().tolist()

    def kept(name, b):
        """Keys or values of sequence b, [H, kv, d]."""
        at = torch.tensor(table[b][:-(-kv[b] // page)], device="cuda")
        if bits8:
            byte = s[name][at].long()
            lookup = torch.cat([_grid(), torch.full((1,), math.nan, dtype=torch.float64, device="cuda")])
            x = torch.where(byte >= 128, -1.0, 1.0) * lookup[byte % 128] * torch.exp2(s[name + "_exp"][at].double() - EXP_BIAS)[..., None]
        else:
            x = s[name][at].double()
        return x.transpose(0, 1).reshape(H, -1, d)[:, :kv[b]]

    if case["op"] == "write":
        out = {}
        for name, rows in (("k", s["K"]), ("v", s["V"])):
            x, pool = rows.double(), torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
            for b, n in enumerate(q):
                position = torch.arange(kv[b] - n, kv[b], device="cuda")
                at = torch.tensor(table[b], device="cuda")[position // page]
                pool[at, :, position % page] = x[:, starts[b]:starts[b + 1]].transpose(0, 1)
            out[name] = pool
        return out
    if case["op"] == "keep":
        return {"K": _value_kept(s["K"].double()) if bits8 else s["K"].double(), "V": _value_kept(s["V"].double()) if bits8 else s["V"].double()}
    if case["op"] == "read":
        return {"K": torch.cat([kept("k", b) for b in range(case["seqs"])], 1), "V": torch.cat([kept("v", b) for b in range(case["seqs"])], 1)}
    G = case["heads"] // H
    out = torch.zeros(s["tokens"], case["heads"] * d, dtype=torch.float64, device="cuda")
    for b, n in enumerate(q):
        K, V = kept("k", b), kept("v", b)
        at = torch.arange(kv[b], device="cuda")
        for lo in range(0, n, 1024):
            hi = min(n, lo + 1024)
            hidden = at[None, :] > (kv[b] - n + torch.arange(lo, hi, device="cuda"))[:, None]
            for h in range(case["heads"]):
                x = s["Q"][h, starts[b] + lo:starts[b] + hi].double() @ K[h // G].T / math.sqrt(d)
                x[hidden] = -math.inf
                out[starts[b] + lo:starts[b] + hi, h * d:(h + 1) * d] = torch.softmax(x, -1) @ V[h // G]
    return out
