"""Operators of a serving step around the paged key/value cache, case by case: the norms before and after a block with its gate and residual scale,
projections with weights of 4 bits and group scales, and the pages of the cache: taken, forked, freed, compacted, copied. `run` computes them as
elementary torch operations, or, where `own` is true, through the package.
"""
import importlib
import math

import torch

own = False

ZERO = 8            # what the code of a weight stands above where there are no zeros


# ---- cases ---------------------------------------------------------------------------------------------------------------------------------
# Norms: rows x d; kind "rms" or "layer"; post: the block's output is normalised too; gate: "none", "row" (one for all rows) or "rows" (one each), through a
# sigmoid where `sigmoid`; bits_x, bits_y: of the residual stream and of the block's output (16: fp16, 32: fp32)
def _norm(name, rows, d, kind, post, gate, sigmoid, bits_x, bits_y):
    return dict(name=name, op="norm", rows=rows, d=d, kind=kind, post=post, gate=gate, sigmoid=sigmoid, bits_x=bits_x, bits_y=bits_y)


# Projections: rows x d_in -> d_out; group: weights to a scale; zeros: a zero point per group; bits_out: 16 (fp16) or 32 (fp32, partial sums of a shard)
def _w4(name, rows, d_in, d_out, group, zeros, bits_out):
    return dict(name=name, op="w4", rows=rows, d_in=d_in, d_out=d_out, group=group, zeros=zeros, bits_out=bits_out)


# Pages: seqs slots, of which `active` have kv_min to kv keys; n: how many children (fork), new sequences of up to q tokens (take), pairs of pages (copy);
# spare: free pages for a hundred in use; the rest as in a paged cache
def _pages(name, op, seqs, active, kv, kv_min, n, q, spare, kv_heads, d_h, page, bits):
    return dict(name=name, op=op, seqs=seqs, active=active, kv=kv, kv_min=kv_min, n=n, q=q, spare=spare, kv_heads=kv_heads, d_h=d_h, page=page, bits=bits)


def listed():
    return [
        # one user's next token between the block and the next one: latency
        _norm("norm_one_token", 1, 4096, "rms", True, "row", False, 16, 16),
        # a prompt of 8192 tokens, a gate for every element
        _norm("norm_prompt", 8192, 4096, "rms", True, "rows", True, 16, 16),
        # a ragged batch, a residual stream and partial sums in fp32, an odd width
        _norm("norm_ragged_f32", 1237, 2049, "layer", False, "none", False, 32, 32),
        # one user's next token through W_O of 32 heads of 128
        _w4("w4_one_token", 1, 4096, 4096, 128, False, 16),
        # a batch's Q, K and V in one, 32 heads of 128 on 8
        _w4("w4_batch_qkv", 16, 4096, 6144, 64, True, 16),
        # a rank's share of W_O of odd size, partial sums
        _w4("w4_odd_shard", 5, 1056, 4163, 32, True, 32),
        # the widest layer, a full batch
        _w4("w4_full_batch", 64, 8192, 32768, 128, False, 16),
        # a second answer to one user's question
        _pages("fork_one", "fork", 8, 1, 1000, 1000, 1, 0, 100, 16, 64, 64, 16),
        # beams of a full batch over 8 bits, tried and dropped
        _pages("fork_beams_8bit", "fork", 256, 48, 8192, 517, 192, 0, 50, 8, 128, 256, 8),
        # new prompts find their pages, and leave
        _pages("take_prompts", "take", 512, 300, 4096, 1, 180, 2048, 150, 8, 64, 16, 16),
        # a fragmented pool
        _pages("compact_pool", "compact", 64, 64, 4096, 333, 0, 0, 60, 8, 128, 64, 16),
        # pages set aside for another pool's use
        _pages("copy_pages_8bit", "copy", 32, 32, 4096, 100, 300, 0, 100, 8, 128, 128, 8),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "w4", "w4", "w4", "fork", "take", "compact", "copy"])
    while True:
        if op == "norm":
            c = _norm("", _log_int(rng, 1, 16384), _log_int(rng, 16, 16384), rng.choice(["rms", "layer"]), rng.random() < 0.5, rng.choice(["none", "row", "rows"]),
                      rng.random() < 0.5, rng.choice([16, 16, 32]), rng.choice([16, 16, 32]))
            fits = c["rows"] * c["d"] <= 3 << 23
        elif op == "w4":
            group = rng.choice([32, 64, 128])
            c = _w4("", _log_int(rng, 1, 64), group * _log_int(rng, 1, 16384 // group), _log_int(rng, 8, 32768), group, rng.random() < 0.5, rng.choice([16, 16, 32]))
            fits = c["d_in"] * c["d_out"] <= 1 << 28
        else:
            kv = _log_int(rng, 1, 8192)
            active = _log_int(rng, 1, 128)
            n = _log_int(rng, 1, 300)
            seqs = active + n if op in ("fork", "take") else active
            c = _pages("", op, seqs, active, kv, _log_int(rng, 1, kv), n if op != "compact" else 0, _log_int(rng, 1, 2048) if op == "take" else 0, rng.randint(20, 150),
                       rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([16, 32, 64, 128, 128]), rng.choice([16, 32, 64, 128, 256]), rng.choice([16, 8]))
            fits = (active * (kv + c["page"]) * (1 + c["spare"] / 100) + n * (c["q"] + c["page"])) * c["kv_heads"] * c["d_h"] <= 3 << 26
        if fits:
            del c["name"]
            return c


def _spread(b, most, fewest):
    """Sequence 0 has the most, the others something in between, each its own."""
    return most if b == 0 else fewest + (most - fewest) * ((b * 40503 + 9973) % 65536) // 65535


def _held(kv, page):
    return -(-kv // page)


def _plan(case):
    """Of the pages' cases, from the sizes alone: keys of every slot, new tokens of every slot, (parent, child) of the forks, pages of the pool."""
    S, A, page = case["seqs"], case["active"], case["page"]
    kv = [_spread(b, case["kv"], case["kv_min"]) if b < A else 0 for b in range(S)]
    forks = [((7 * i + i // A) % A, A + i) for i in range(case["n"])] if case["op"] == "fork" else []
    new = [_spread(b - A, case["q"], 1) if A <= b < A + case["n"] else 0 for b in range(S)] if case["op"] == "take" else [0] * S
    used = sum(_held(n, page) for n in kv)
    most = max([_held(n, page) for n in kv] + [_held(n, page) for n in new])
    want = sum(_held(n, page) for n in new) + len(forks) + (case["n"] if case["op"] == "copy" else 0)
    return kv, new, forks, used, used + max(want, used * case["spare"] // 100) + 3, most


def work(case):
    if case["op"] == "norm":
        n, d = case["rows"], case["d"]
        vectors = (4 if case["kind"] == "layer" else 2) if case["post"] else (2 if case["kind"] == "layer" else 1)
        each = 2 * case["bits_x"] // 8 + case["bits_y"] // 8 + 2 + (2 if case["gate"] == "rows" else 0)
        return {"bytes": n * d * each + 2 * d * (vectors + (case["gate"] == "row")), "flops": 12 * n * d}
    if case["op"] == "w4":
        n, k, m = case["rows"], case["d_in"], case["d_out"]
        return {"bytes": k * m // 2 + k // case["group"] * m * (3 if case["zeros"] else 2) + n * (2 * k + m * case["bits_out"] // 8), "flops": 2 * n * k * m}
    kv, new, forks, used, pool, most = _plan(case)
    key = 2 * case["kv_heads"] * (case["d_h"] * (2 if case["bits"] == 16 else 1) + (1 if case["bits"] == 8 else 0))      # bytes of a key in the cache
    page = key * case["page"]
    if case["op"] == "fork":       # the last pages' keys twice, refs, the children's entries: written, read once more to be freed, and the parents' read
        entries = sum(_held(kv[p], case["page"]) for p, _ in forks)
        return {"bytes": 2 * key * sum(kv[p] % case["page"] for p, _ in forks) + 4 * pool + 4 * 5 * entries, "flops": 0}
    if case["op"] == "take":       # refs; entries and counts of new pages written, read and written when they are freed
        return {"bytes": 4 * pool + 4 * 5 * sum(_held(n, case["page"]) for n in new), "flops": 0}
    if case["op"] == "compact":    # about as many pages move as there are free ones among the first `used`
        moved = used * (pool - used) // pool
        return {"bytes": 2 * page * moved + 4 * 3 * pool + 4 * 2 * used, "flops": 0}
    return {"bytes": case["n"] * (2 * page + 8), "flops": 0}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 29)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    def real(bits):
        return torch.float16 if bits == 16 else torch.float32

    s = {"case": case}
    if case["op"] == "norm":
        n, d = case["rows"], case["d"]
        loud = torch.where(torch.rand(d, generator=gen, device="cuda") < 0.01, 20.0, 1.0)         # a few channels of a residual stream are far above the others
        s["x"], s["y"] = (2 * loud * normal(n, d) + 0.1).to(real(case["bits_x"])), normal(n, d).to(real(case["bits_y"]))
        s["gate"] = None if case["gate"] == "none" else normal(n if case["gate"] == "rows" else 1, d).half()
        for name in ("post", "pre"):
            there = name == "pre" or case["post"]
            s[name + "_w"] = (1 + 0.2 * normal(d)).half() if there else None
            s[name + "_b"] = (0.1 * normal(d)).half() if there and case["kind"] == "layer" else None
        s["residual_scale"], s["block_scale"], s["eps"] = 0.9375, 0.5, 1e-5
        s["x_out"], s["h"] = torch.zeros_like(s["x"]), torch.zeros(n, d, dtype=torch.float16, device="cuda")
        return s
    if case["op"] == "w4":
        n, k, m, groups = case["rows"], case["d_in"], case["d_out"], case["d_in"] // case["group"]
        s["codes"] = torch.randint(0, 256, (m, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        s["scales"] = ((0.5 + torch.rand(groups, m, generator=gen, device="cuda")) * (0.25 / math.sqrt(k))).half()
        s["zeros"] = torch.randint(5, 12, (groups, m), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        s["X"] = normal(n, k).half()
        s["out"] = torch.zeros(n, m, dtype=real(case["bits_out"]), device="cuda")
        return s
    kv, new, forks, used, pool, most = _plan(case)
    H, d, page = case["kv_heads"], case["d_h"], case["page"]
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table, refs, at = torch.zeros(case["seqs"], most, dtype=torch.int64), torch.zeros(pool, dtype=torch.int32, device="cuda"), 0
    held = torch.zeros(case["seqs"], most, dtype=torch.bool)
    for b, n in enumerate(kv):
        m = _held(n, page)
        table[b, :m], held[b, :m] = torch.arange(at, at + m), True
        at += m
    refs[order[:used].long()] = 1
    s["refs"], s["kv_len"] = refs, torch.tensor(kv, dtype=torch.int32).cuda()
    s["pages"] = torch.where(held.cuda(), order[table.cuda()], 0).to(torch.int32)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["q_start"] = torch.tensor(starts, dtype=torch.int32).cuda()
    if forks:
        s["parents"], s["children"] = (torch.tensor(x, dtype=torch.int32).cuda() for x in zip(*forks))
    if case["op"] == "take":
        s["leave"] = torch.arange(case["active"], case["active"] + case["n"], dtype=torch.int32, device="cuda")
        return s
    if case["op"] == "copy":
        n = min(case["n"], used)
        s["src"], s["dst"] = order[:n].clone(), order[used:used + n].clone()
    if case["op"] == "compact":
        s["pages_out"], s["refs_out"], s["moved"] = (torch.zeros_like(x) for x in (s["pages"], refs, refs))
    for name in ("k", "v"):
        if case["bits"] == 16:
            s[name] = torch.randn(pool, H, page, d, generator=gen, device="cuda", dtype=torch.float16)
        else:
            code = torch.randint(0, 254, (pool, H, page, d), generator=gen, device="cuda", dtype=torch.uint8)
            s[name] = torch.where(code >= 127, code + 1, code)                                    # 127 and 255 are NaN
            s[name + "_exp"] = torch.randint(110, 130, (pool, H, page), generator=gen, device="cuda", dtype=torch.uint8)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------------------
def _normalised(v, kind, eps, w, b):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w.float()
    return v if b is None else v + b.float()


def _block_norm(s):
    c = s["case"]
    n = s["y"].float()
    if c["post"]:
        n = _normalised(n, c["kind"], s["eps"], s["post_w"], s["post_b"])
    if s["gate"] is not None:
        g = s["gate"].float()
        n = n * (torch.sigmoid(g) if c["sigmoid"] else g)
    r = s["residual_scale"] * s["x"].float() + s["block_scale"] * n
    return {"x_out": r.to(s["x"].dtype), "h": _normalised(r, c["kind"], s["eps"], s["pre_w"], s["pre_b"]).half()}


def _project_w4(s):
    c = s["case"]
    out = torch.empty_like(s["out"])
    X, step = s["X"].float(), max(1, (1 << 26) // c["d_in"])
    for lo in range(0, c["d_out"], step):
        codes = s["codes"][lo:lo + step]
        q = torch.stack([codes & 15, codes >> 4], -1).reshape(len(codes), -1, c["group"]).float()
        zero = ZERO if s["zeros"] is None else s["zeros"][:, lo:lo + step].t().float().unsqueeze(-1)
        W = ((q - zero) * s["scales"][:, lo:lo + step].t().float().unsqueeze(-1)).reshape(len(codes), -1)
        out[:, lo:lo + step] = (X @ W.t()).to(out.dtype)
    return out


def _page_count(kv, page):
    return torch.div(kv + (page - 1), page, rounding_mode="floor")


def _free_pages(refs):
    """All pages, the free ones first, lowest first."""
    return torch.argsort((refs > 0).to(torch.uint8), stable=True)


def _release(s, seqs):
    seqs, page = seqs.long(), s["case"]["page"]
    entry = torch.arange(s["pages"].shape[1], device="cuda")
    held = entry < _page_count(s["kv_len"][seqs], page)[:, None]
    at = s["pages"][seqs].long()
    s["refs"].index_add_(0, at.reshape(-1), held.reshape(-1).to(torch.int32), alpha=-1)
    s["kv_len"][seqs] = 0


def _take(s):
    page, refs, kv = s["case"]["page"], s["refs"], s["kv_len"]
    after = kv + s["q_start"][1:] - s["q_start"][:-1]
    have, want = _page_count(kv, page).long(), _page_count(after, page).long()
    need = want - have
    before = need.cumsum(0) - need
    entry = torch.arange(s["pages"].shape[1], device="cuda")
    fresh = (entry >= have[:, None]) & (entry < want[:, None])
    free = _free_pages(refs)
    rank = (before[:, None] + entry - have[:, None]).clamp(0, len(refs) - 1)
    s["pages"].copy_(torch.where(fresh, free[rank].to(torch.int32), s["pages"]))
    refs[free] = torch.where(torch.arange(len(refs), device="cuda") < need.sum(), 1, refs[free])
    kv.copy_(after)


def _cache_parts(s):
    return [s[x] for x in ("k", "v", "k_exp", "v_exp") if x in s]


def _fork(s):
    page, refs, kv, pages = s["case"]["page"], s["refs"], s["kv_len"], s["pages"]
    parents, children = s["parents"].long(), s["children"].long()
    n, rest = kv[parents], kv[parents] % page
    full = torch.div(n, page, rounding_mode="floor").long()
    partly = rest > 0
    rank = partly.long().cumsum(0) - partly.long()
    fresh = _free_pages(refs)[rank.clamp(max=len(refs) - 1)]
    entry = torch.arange(pages.shape[1], device="cuda")
    at = pages[parents]
    shared, last = entry < full[:, None], (entry == full[:, None]) & partly[:, None]
    source = torch.gather(at, 1, full.clamp(max=pages.shape[1] - 1)[:, None]).squeeze(1).long()
    pages[children] = torch.where(shared, at, torch.where(last, fresh[:, None].to(torch.int32), pages[children]))
    refs.index_add_(0, at.long().reshape(-1), shared.reshape(-1).to(torch.int32))
    refs.index_add_(0, fresh, partly.to(torch.int32))
    kv[children] = n
    who = torch.nonzero(partly).squeeze(1)
    source, target, rest = source[who], fresh[who], rest[who]
    for x in _cache_parts(s):
        there = torch.arange(page, device="cuda") < rest[:, None]
        there = there.reshape(len(rest), 1, page, *[1] * (x.dim() - 3))
        x[target] = torch.where(there, x[source], x[target])


def _compact(s):
    page, refs, kv, pages = s["case"]["page"], s["refs"], s["kv_len"], s["pages"]
    used, index = refs > 0, torch.arange(len(refs), device="cuda")
    live = used.sum()
    movers, holes = torch.nonzero(used & (index >= live)).squeeze(1), torch.nonzero(~used & (index < live)).squeeze(1)
    moved = torch.where(used, index, -1)
    moved[movers] = holes
    s["moved"].copy_(moved)
    s["refs_out"].zero_()
    s["refs_out"][moved[used]] = refs[used]
    held = torch.arange(pages.shape[1], device="cuda") < _page_count(kv, page)[:, None]
    s["pages_out"].copy_(torch.where(held, moved[pages.long()].to(torch.int32), s["pages_out"]))
    for x in _cache_parts(s):
        x[holes] = x[movers]


# ---- through the package -------------------------------------------------------------------------------------------------------------------
class _Call:
    """What a program keeps for its calls: the package's descriptions of its tensors, and a workspace."""

    def __init__(self, s):
        c, self.pkg = s["case"], importlib.import_module("eager-flash-attention_b200")
        pkg, op = self.pkg, c["op"]
        self.device = torch.cuda.current_device()
        if op == "norm":
            self.how = pkg.block_norm_params(c["d"], kind=pkg.NORM_RMS if c["kind"] == "rms" else pkg.NORM_LAYER, eps=s["eps"], post=c["post"], pre=True,
                                             gate=pkg.GATE_NONE if c["gate"] == "none" else pkg.GATE_SIGMOID if c["sigmoid"] else pkg.GATE_PLAIN,
                                             gate_rows=c["gate"] == "rows", residual_scale=s["residual_scale"], block_scale=s["block_scale"],
                                             x_dtype=pkg.F16 if c["bits_x"] == 16 else pkg.F32, y_dtype=pkg.F16 if c["bits_y"] == 16 else pkg.F32)
        elif op == "w4":
            self.weight = pkg.w4_weight(s["codes"], s["scales"], s["zeros"])
        else:
            self.pool = pkg.page_pool(s["refs"], s["pages"], s["kv_len"], c["page"])
            if "k" in s:
                self.cache = pkg.paged_cache(s["k"], s["v"], s.get("k_exp"), s.get("v_exp"))
            size = pkg.pages_workspace(self.pool) if op != "copy" else 0
            self.workspace = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None


def _through_package(s):
    call = s.get("call")
    if call is None:
        call = s["call"] = _Call(s)
    pkg, op, stream = call.pkg, s["case"]["op"], torch._C._cuda_getCurrentRawStream(call.device)    # the current stream, without 3 us for an object of it
    if op == "norm":
        pkg.block_norm(s["x"], s["y"], s["x_out"], s["h"], s["case"]["rows"], call.how, s["gate"], s["post_w"], s["post_b"], s["pre_w"], s["pre_b"], stream=stream)
    elif op == "w4":
        pkg.project_w4(s["X"], call.weight, s["out"], s["case"]["rows"], stream=stream)
    elif op == "take":
        pkg.pages_take(call.pool, s["q_start"], call.workspace, stream=stream)
        pkg.pages_free(call.pool, s["leave"], stream=stream)
    elif op == "fork":
        pkg.pages_fork(call.pool, call.cache, s["parents"], s["children"], call.workspace, stream=stream)
        pkg.pages_free(call.pool, s["children"], stream=stream)
    elif op == "compact":
        pkg.pages_compact(call.pool, call.cache, s["pages_out"], s["refs_out"], s["moved"], call.workspace, stream=stream)
    else:
        pkg.pages_copy(call.cache, s["src"], s["dst"], stream=stream)


def _values(s):
    """The cache's contents: fp16, or the codes as the numbers they are and their exponents' bytes."""
    out = {x: s[x] if s["case"]["bits"] == 16 else s[x].view(torch.float8_e4m3fn) for x in ("k", "v")}
    return {**out, **{x: s[x] for x in ("k_exp", "v_exp") if x in s}}


def run(state):
    op = state["case"]["op"]
    if own:
        _through_package(state)
        if op == "norm":
            return {"x_out": state["x_out"], "h": state["h"]}
        if op == "w4":
            return state["out"]
    elif op == "norm":
        return _block_norm(state)
    elif op == "w4":
        return _project_w4(state)
    elif op == "take":
        _take(state)
        _release(state, state["leave"])
    elif op == "fork":
        _fork(state)
        _release(state, state["children"])
    elif op == "compact":
        _compact(state)
    else:
        for x in _cache_parts(state):
            x[state["dst"].long()] = x[state["src"].long()]
    if op == "copy":
        return _values(state)
    if op == "compact":
        return {**_values(state), "pages": state["pages_out"], "refs": state["refs_out"], "moved": state["moved"]}
    return {**(_values(state) if op == "fork" else {}), **{x: state[x] for x in ("pages", "refs", "kv_len")}}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------------
def _exact_norm(s):
    c, eps = s["case"], s["eps"]
    x_out, h = torch.empty(c["rows"], c["d"], dtype=torch.float64, device="cuda"), torch.empty(c["rows"], c["d"], dtype=torch.float64, device="cuda")

    def norm(v, w, b):
        centre = torch.sum(v, -1, keepdim=True) / c["d"] if c["kind"] == "layer" else torch.zeros_like(v[:, :1])
        power = torch.sum((v - centre) ** 2, -1, keepdim=True) / c["d"]
        v = (v - centre) / torch.sqrt(power + eps) * w.double()
        return v if b is None else v + b.double()

    for lo in range(0, c["rows"], 1024):
        at = slice(lo, lo + 1024)
        n = s["y"][at].double()
        n = norm(n, s["post_w"], s["post_b"]) if c["post"] else n
        if s["gate"] is not None:
            g = (s["gate"][at] if c["gate"] == "rows" else s["gate"]).double()
            n = n / (1 + torch.exp(-g)) if c["sigmoid"] else n * g
        r = s["x"][at].double() * s["residual_scale"] + n * s["block_scale"]
        x_out[at], h[at] = r, norm(r, s["pre_w"], s["pre_b"])
    return {"x_out": x_out, "h": h}


def _exact_w4(s):
    c = s["case"]
    out = torch.empty(c["rows"], c["d_out"], dtype=torch.float64, device="cuda")
    for lo in range(0, c["d_out"], 2048):
        hi, total = min(c["d_out"], lo + 2048), 0
        for g in range(c["d_in"] // c["group"]):
            k = slice(g * c["group"], (g + 1) * c["group"])
            byte = s["codes"][lo:hi, k.start // 2:k.stop // 2].double()
            high = torch.floor(byte / 16)
            w = torch.empty(hi - lo, c["group"], dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = byte - 16 * high, high
            w -= ZERO if s["zeros"] is None else s["zeros"][g, lo:hi, None].double()
            total = total + (s["X"][:, k].double() @ w.T) * s["scales"][g, lo:hi].double()
        out[:, lo:hi] = total
    return out


def _exact_pages(s):
    """The lists as lists, one sequence and one page after another."""
    c, page = s["case"], s["case"]["page"]
    refs, table, kv = s["refs"].tolist(), s["pages"].tolist(), s["kv_len"].tolist()
    data = {x: s[x].clone() for x in ("k", "v", "k_exp", "v_exp") if x in s}
    pairs = []                                                              # (from, to, keys)

    def lowest_free():
        return refs.index(0)

    def leave(b):
        for i in range(-(-kv[b] // page)):
            refs[table[b][i]] -= 1
        kv[b] = 0

    out = {}
    if c["op"] == "take":
        starts = s["q_start"].tolist()
        for b in range(c["seqs"]):
            for key in range(kv[b], kv[b] + starts[b + 1] - starts[b]):
                if key % page == 0:
                    table[b][key // page] = lowest_free()
                    refs[table[b][key // page]] = 1
            kv[b] += starts[b + 1] - starts[b]
        for b in s["leave"].tolist():
            leave(b)
    elif c["op"] == "fork":
        for p, b in zip(s["parents"].tolist(), s["children"].tolist()):
            for i in range(kv[p] // page):
                table[b][i] = table[p][i]
                refs[table[p][i]] += 1
            if kv[p] % page:
                i = kv[p] // page
                table[b][i] = lowest_free()
                refs[table[b][i]] = 1
                pairs.append((table[p][i], table[b][i], kv[p] % page))
            kv[b] = kv[p]
        for b in s["children"].tolist():
            leave(b)
    elif c["op"] == "compact":
        live = sum(r > 0 for r in refs)
        holes = [p for p in range(live) if refs[p] == 0]
        movers = [p for p in range(live, len(refs)) if refs[p] > 0]
        to = {p: p for p in range(len(refs)) if refs[p] > 0}
        to.update(zip(movers, holes))
        pairs = [(p, q, page) for p, q in zip(movers, holes)]
        out["moved"] = [to.get(p, -1) for p in range(len(refs))]
        new_refs, new_table = [0] * len(refs), s["pages_out"].tolist()
        for p, q in to.items():
            new_refs[q] = refs[p]
        for b, n in enumerate(kv):
            for i in range(-(-n // page)):
                new_table[b][i] = to[table[b][i]]
        refs, table = new_refs, new_table
    else:
        pairs = [(p, q, page) for p, q in zip(s["src"].tolist(), s["dst"].tolist())]
    for name, x in data.items():
        for p, q, n in pairs:
            x[q, :, :n] = x[p, :, :n]
    if data:
        out.update({x: (data[x] if c["bits"] == 16 else data[x].view(torch.float8_e4m3fn)).double() for x in ("k", "v")})
        out.update({x: data[x] for x in ("k_exp", "v_exp") if x in data})
    if c["op"] != "copy":
        out.update(pages=torch.tensor(table, dtype=torch.int32).cuda(), refs=torch.tensor(refs, dtype=torch.int32).cuda())
        if c["op"] == "compact":
            out["moved"] = torch.tensor(out["moved"], dtype=torch.int32).cuda()
        else:
            out["kv_len"] = torch.tensor(kv, dtype=torch.int32).cuda()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if case["op"] == "norm" else _exact_w4(s) if case["op"] == "w4" else _exact_pages(s)
