"""A pool of pages as lists, one slot and one page after another: what the page operators have to give."""
import torch


class Model:
    """refs, pages and kv_len on the host."""

    def __init__(self, num_pages, page, num_seqs, max_pages):
        self.page, self.max_pages = page, max_pages
        self.refs, self.kv = [0] * num_pages, [0] * num_seqs
        self.pages = [[-7] * max_pages for _ in range(num_seqs)]
        self.wrong = False                                 # something was to be reported

    def held(self, b):
        return -(-self.kv[b] // self.page)

    def _free(self):
        for p, n in enumerate(self.refs):
            if n <= 0:
                self.refs[p] = 1
                return p
        self.wrong = True
        return -1

    def take(self, new):
        for b, n in enumerate(new):
            after = min(self.kv[b] + max(n, 0), self.max_pages * self.page)
            self.wrong |= after != self.kv[b] + n
            for e in range(self.held(b), -(-after // self.page)):
                self.pages[b][e] = self._free()
            self.kv[b] = after

    def fork(self, parents, children):
        """Pairs (from, to, keys) that were copied."""
        before, named, moves = [list(r) for r in self.pages], set(), []
        kv = list(self.kv)
        for p, c in zip(parents, children):
            S = len(kv)
            first = c not in named
            named.add(c)
            if not (0 <= c < S and 0 <= p < S and first and kv[c] == 0):
                self.wrong = True
                continue
            full, rest = divmod(kv[p], self.page)
            for e in range(full):
                self.pages[c][e] = before[p][e]
                if before[p][e] >= 0:
                    self.refs[before[p][e]] += 1
                else:
                    self.wrong = True
            if rest:
                source = before[p][full]
                if source < 0:
                    self.wrong = True
                self.pages[c][full] = self._free() if source >= 0 else -1
                if self.pages[c][full] >= 0:
                    moves.append((source, self.pages[c][full], rest))
            self.kv[c] = kv[p]
        return moves

    def free(self, seqs):
        for b in seqs:
            if not 0 <= b < len(self.kv):
                self.wrong = True
                continue
            for e in range(self.held(b)):
                if self.pages[b][e] >= 0:
                    self.refs[self.pages[b][e]] -= 1
            self.kv[b] = 0

    def compact(self):
        """(pages, refs, moved, pairs (from, to)) after the moves; entries that are not written stay as they are here."""
        live = sum(n > 0 for n in self.refs)
        holes, movers = [p for p in range(live) if self.refs[p] <= 0], [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        moved = [p if n > 0 else -1 for p, n in enumerate(self.refs)]
        for p, q in zip(movers, holes):
            moved[p] = q
        refs = [0] * len(self.refs)
        for p, q in enumerate(moved):
            if q >= 0:
                refs[q] = self.refs[p]
        pages = [list(r) for r in self.pages]
        for b in range(len(self.kv)):
            for e in range(self.held(b)):
                pages[b][e] = moved[pages[b][e]] if pages[b][e] >= 0 else -1
        return pages, refs, moved, list(zip(movers, holes))


class Device:
    """The same on the GPU, with a cache of random contents."""

    def __init__(self, pkg, num_pages, page, num_seqs, max_pages, H=2, d=16, bits=16, gap=0, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.pkg = pkg
        self.refs = torch.zeros(num_pages, dtype=torch.int32, device="cuda")
        self.pages = torch.full((num_seqs, max_pages), -7, dtype=torch.int32, device="cuda")
        self.kv = torch.zeros(num_seqs, dtype=torch.int32, device="cuda")
        n = H * page * d
        def one():
            store = torch.randint(0, 256, (num_pages, (n + gap) * (bits // 8)), generator=gen, device="cuda", dtype=torch.uint8)
            store = store.view(torch.float16) if bits == 16 else store
            return store.as_strided((num_pages, H, page, d), (n + gap, page * d, d, 1))
        self.parts = [one(), one()]
        if bits == 8:
            self.parts += [torch.randint(0, 256, (num_pages, H, page), generator=gen, device="cuda", dtype=torch.uint8) for _ in range(2)]
        self.cache = pkg.paged_cache(*self.parts)
        self.pool = pkg.page_pool(self.refs, self.pages, self.kv, page)
        self.ws = torch.full((pkg.pages_workspace(self.pool),), 0xA5, dtype=torch.uint8, device="cuda")

    def bits(self):
        """All contents as whole numbers, copies."""
        return [x.contiguous().view(torch.int16) if x.dtype == torch.float16 else x.clone() for x in self.parts]

    def ints(self, *x):
        return torch.tensor(list(x), dtype=torch.int32, device="cuda")

    def starts(self, new, first=0):
        at = [first]
        for n in new:
            at.append(at[-1] + n)
        return self.ints(*at)

    def load(self, m):
        self.refs.copy_(torch.tensor(m.refs, dtype=torch.int32))
        self.pages.copy_(torch.tensor(m.pages, dtype=torch.int32).reshape(self.pages.shape))
        self.kv.copy_(torch.tensor(m.kv, dtype=torch.int32))

    def same(self, m):
        torch.cuda.synchronize()
        assert self.kv.tolist() == m.kv
        assert self.refs.tolist() == m.refs
        assert self.pages.tolist() == m.pages


def moved_bits(before, moves):
    """Contents after (from, to, keys): the first keys of a page."""
    after = [x.clone() for x in before]
    for p, q, n in moves:
        for x, y in zip(after, before):
            x[q, :, :n] = y[p, :, :n]
    return after


def equal_bits(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))
