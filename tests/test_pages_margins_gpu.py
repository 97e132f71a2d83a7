"""Pools whose arrays hold what they should not: every array stands between margins that have to stay, what a call leaves is compared entry by entry with the list of what it
should, and what it reports is the one thing that is wrong."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

BIG, MARGIN, MARK = 2 ** 31 - 1, 96, -559038737
BAD_PAGE, BAD_LENGTH, NO_PAGE, BAD_SLOT = 2, 3, 4, 5
TAKE, FORK, FREE, COMPACT = 60, 61, 62, 63


class Pool:
    """A pool, its cache and a workspace of just the size that is asked for, each between margins."""

    def __init__(self, pkg, num_pages, page, num_seqs, max_pages, H=2, d=16):
        pkg.kernel_status_reset()
        self.pkg, self.page, self.cap = pkg, page, page * max_pages
        self.stores = []
        self.refs, self.kv = self.ints([0] * num_pages), self.ints([0] * num_seqs)
        self.pages = self.ints([-7] * (num_seqs * max_pages)).view(num_seqs, max_pages)
        self.pool = pkg.page_pool(self.refs, self.pages, self.kv, page)
        self.ws = self.ints([0x5A5A5A5A] * (pkg.pages_workspace(self.pool) // 4))
        gen = torch.Generator(device="cuda").manual_seed(num_pages)
        self.whole = [torch.randint(-30000, 30000, (num_pages + 2, H, page, d), generator=gen, device="cuda", dtype=torch.int16).view(torch.float16) for _ in range(2)]
        self.before = [x.clone() for x in self.whole]
        self.cache = pkg.paged_cache(*(x[1:-1] for x in self.whole))

    def ints(self, values):
        n = len(values)
        store = torch.full((n + 2 * MARGIN,), MARK, dtype=torch.int32, device="cuda")
        store[MARGIN:MARGIN + n] = torch.tensor(values, dtype=torch.int32, device="cuda")
        self.stores.append((store, n))
        return store[MARGIN:MARGIN + n]

    def put(self, refs=None, pages=None, kv=None):
        for x, y in ((self.refs, refs), (self.pages, pages), (self.kv, kv)):
            if y is not None:
                x.copy_(torch.tensor(y, dtype=torch.int32))

    def margins(self):
        torch.cuda.synchronize()
        for store, n in self.stores:
            assert torch.all(store[:MARGIN] == MARK) and torch.all(store[MARGIN + n:] == MARK)
        for x, y in zip(self.whole, self.before):
            for end in (0, -1):
                assert torch.equal(x[end].view(torch.int16), y[end].view(torch.int16))

    def moved(self, moves):
        """The cache's contents: those of before with (from, to, keys) moved."""
        for x, y in zip(self.whole, self.before):
            want = y.clone()
            for p, q, n in moves:
                want[1 + q, :, :n] = y[1 + p, :, :n]
            assert torch.equal(x.view(torch.int16), want.view(torch.int16))

    def expect(self, refs, pages, kv, code, site, who=None):
        self.margins()
        assert self.kv.tolist() == kv
        assert self.refs.tolist() == refs
        assert self.pages.tolist() == pages
        status = self.pkg.kernel_status()
        assert status[0] == code and (code == 0 or status[2] == site) and (who is None or status[1] == who), tuple(status)


def pool(pkg):
    """Slots of 20, 40, 64 and 5 keys in pages 0 to 9 of 16, four to a slot; two more slots; 14 pages."""
    p = Pool(pkg, 14, 16, 6, 4)
    refs, kv = [1] * 10 + [0] * 4, [20, 40, 64, 5, 0, 0]
    pages = [[0, 1, -7, -7], [2, 3, 4, -7], [5, 6, 7, 8], [9, -7, -7, -7], [-7] * 4, [-7] * 4]
    p.put(refs, pages, kv)
    return p, refs, pages, kv


# ---- take ----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("slot,wrong,add,after", [(1, BIG, 0, 64), (1, BIG, 5, 64), (1, 65, 0, 64), (4, -1, 0, 0), (4, -BIG - 1, 20, 20), (4, -5, 3, 3)])
def test_take_from_a_length_outside_the_table(pkg, torch_cuda, slot, wrong, add, after):
    p, refs, pages, kv = pool(pkg)
    p.put(kv=kv[:slot] + [wrong] + kv[slot + 1:])
    starts = p.ints([7] * (slot + 1) + [7 + add] * (6 - slot))
    pkg.pages_take(p.pool, starts, p.ws)
    kv[slot] = after
    if slot == 4:
        for e in range(-(-after // 16)):
            pages[4][e], refs[10 + e] = 10 + e, 1
    p.expect(refs, pages, kv, BAD_LENGTH, TAKE, slot)


@pytest.mark.parametrize("starts,after", [([0, 0, 0, 0, -3, -3, -3], 5), ([0, 0, 0, 0, 100, 100, 100], 64), ([0, 0, 0, 0, BIG, BIG, BIG], 64),
                                          ([BIG, BIG, BIG, BIG, -BIG, -BIG, -BIG], 5), ([-BIG, -BIG, -BIG, -BIG, BIG, BIG, BIG], 64)])
def test_take_of_more_or_fewer_tokens_than_there_can_be(pkg, torch_cuda, starts, after):
    p, refs, pages, kv = pool(pkg)
    pkg.pages_take(p.pool, p.ints(starts), p.ws)
    kv[3] = after
    for e in range(1, -(-after // 16)):
        pages[3][e], refs[9 + e] = 9 + e, 1
    p.expect(refs, pages, kv, BAD_LENGTH, TAKE, 3)


def test_take_of_the_last_pages_and_one_more(pkg, torch_cuda):
    p, refs, pages, kv = pool(pkg)
    pkg.pages_take(p.pool, p.ints([0, 0, 0, 0, 0, 64, 64]), p.ws)
    pages[4], kv[4], refs = [10, 11, 12, 13], 64, [1] * 14
    p.expect(refs, pages, kv, 0, TAKE)
    pkg.pages_take(p.pool, p.ints([0, 0, 9, 9, 9, 9, 9]), p.ws)                    # 40 + 9 keys: a page that there is not
    pages[1][3], kv[1] = -1, 49
    p.expect(refs, pages, kv, NO_PAGE, TAKE, 1)
    p.moved([])


# ---- fork ----------------------------------------------------------------------------------------------------------------------------------
def test_fork_of_a_parent_with_too_many_keys(pkg, torch_cuda):
    p, refs, pages, kv = pool(pkg)
    kv[2] = BIG
    p.put(kv=kv)
    pkg.pages_fork(p.pool, p.cache, p.ints([2]), p.ints([5]), p.ws)
    kv[5], pages[5] = 64, list(pages[2])
    for q in pages[2]:
        refs[q] = 2
    p.expect(refs, pages, kv, BAD_LENGTH, FORK, 2)
    p.moved([])


@pytest.mark.parametrize("wrong", [14, BIG, -BIG - 1, -2, -1])
@pytest.mark.parametrize("entry", [0, 1, 2])
def test_fork_of_a_parent_with_a_page_outside_the_pool(pkg, torch_cuda, wrong, entry):
    """A full page, or the last one: the child has none there. -1, of a parent that got no page, is reported too."""
    p, refs, pages, kv = pool(pkg)
    pages[1][entry] = wrong
    p.put(pages=pages)
    pkg.pages_fork(p.pool, p.cache, p.ints([1]), p.ints([4]), p.ws)
    kv[4] = 40
    for e in range(2):
        pages[4][e] = pages[1][e] if e != entry else -1
        if e != entry:
            refs[pages[1][e]] = 2
    pages[4][2] = -1 if entry == 2 else 10
    refs[10] = 0 if entry == 2 else 1
    p.expect(refs, pages, kv, BAD_PAGE, FORK, 1)
    p.moved([] if entry == 2 else [(4, 10, 8)])


@pytest.mark.parametrize("parent,child,who", [(0, 6, 0), (0, -1, 0), (0, BIG, 0), (0, -BIG - 1, 0), (6, 4, 4), (-1, 4, 4), (BIG, 5, 5), (0, 1, 1)])
def test_fork_of_a_slot_that_there_is_not(pkg, torch_cuda, parent, child, who):
    p, refs, pages, kv = pool(pkg)
    pkg.pages_fork(p.pool, p.cache, p.ints([parent]), p.ints([child]), p.ws)
    p.expect(refs, pages, kv, BAD_SLOT, FORK, who)
    p.moved([])


# ---- free ----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("slot,wrong", [(2, BIG), (2, 65), (0, -1), (0, -BIG - 1)])
def test_free_of_a_length_outside_the_table(pkg, torch_cuda, slot, wrong):
    p, refs, pages, kv = pool(pkg)
    p.put(kv=kv[:slot] + [wrong] + kv[slot + 1:])
    pkg.pages_free(p.pool, p.ints([slot]))
    kv[slot] = 0
    if slot == 2:
        refs[5:9] = [0] * 4
    p.expect(refs, pages, kv, BAD_LENGTH, FREE, slot)


@pytest.mark.parametrize("wrong,code", [(14, BAD_PAGE), (BIG, BAD_PAGE), (-BIG - 1, BAD_PAGE), (-2, BAD_PAGE), (-1, 0)])
def test_free_of_a_page_outside_the_pool(pkg, torch_cuda, wrong, code):
    p, refs, pages, kv = pool(pkg)
    pages[1][1] = wrong
    p.put(pages=pages)
    pkg.pages_free(p.pool, p.ints([1, 1]))
    kv[1], refs[2], refs[4] = 0, 0, 0
    p.expect(refs, pages, kv, code, FREE, 1 if code else None)


@pytest.mark.parametrize("seqs,place", [([6], 0), ([0, -1], 1), ([0, BIG], 1), ([-BIG - 1, 0], 0)])
def test_free_of_a_slot_that_there_is_not(pkg, torch_cuda, seqs, place):
    p, refs, pages, kv = pool(pkg)
    pkg.pages_free(p.pool, p.ints(seqs))
    if 0 in seqs:
        kv[0], refs[0], refs[1] = 0, 0, 0
    p.expect(refs, pages, kv, BAD_SLOT, FREE, place)


# ---- compact -------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("wrong,code", [(14, BAD_PAGE), (BIG, BAD_PAGE), (-BIG - 1, BAD_PAGE), (-2, BAD_PAGE), (-1, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact_with_a_page_outside_the_pool(pkg, torch_cuda, wrong, code, in_place):
    """Slot 0 gone: pages 8 and 9 move to 0 and 1. The entry has no page after that."""
    p, refs, pages, kv = pool(pkg)
    kv[0], refs[0], refs[1], pages[1][1], refs[3] = 0, 0, 0, wrong, 0                  # pages 0, 1 and 3 are free: 7 in use
    p.put(refs, pages, kv)
    out = (p.pages, p.refs) if in_place else (p.ints([-9] * 24).view(6, 4), p.ints([-9] * 14))
    moved = p.ints([-9] * 14)
    pkg.pages_compact(p.pool, p.cache, *out, moved, p.ws)
    new = {2: 2, 4: 4, 5: 5, 6: 6, 7: 0, 8: 1, 9: 3}
    want = [[-7] * 4 if in_place else [-9] * 4 for _ in range(6)]
    if in_place:
        want = [list(r) for r in pages]
    for b, held in ((1, 3), (2, 4), (3, 1)):
        for e in range(held):
            want[b][e] = new.get(pages[b][e], -1)
    new_refs = [1 if q in new.values() else 0 for q in range(14)]
    p.expect(*((new_refs, want) if in_place else (refs, pages)), kv, code, COMPACT, 1 if code else None)
    assert out[0].tolist() == want and out[1].tolist() == new_refs and moved.tolist() == [new.get(q, -1) for q in range(14)]
    p.moved([(7, 0, 16), (8, 1, 16), (9, 3, 16)])


@pytest.mark.parametrize("slot,wrong,held", [(2, BIG, 4), (4, -1, 0), (4, -BIG - 1, 0)])
def test_compact_with_a_length_outside_the_table(pkg, torch_cuda, slot, wrong, held):
    p, refs, pages, kv = pool(pkg)
    kv[slot] = wrong
    p.put(kv=kv)
    pages_out, refs_out, moved = p.ints([-9] * 24).view(6, 4), p.ints([-9] * 14), p.ints([-9] * 14)
    pkg.pages_compact(p.pool, p.cache, pages_out, refs_out, moved, p.ws)
    p.expect(refs, pages, kv, BAD_LENGTH, COMPACT, slot)
    assert pages_out.tolist() == [[0, 1, -9, -9], [2, 3, 4, -9], [5, 6, 7, 8], [9, -9, -9, -9], [-9] * 4, [-9] * 4]
    assert refs_out.tolist() == refs and moved.tolist() == list(range(10)) + [-1] * 4


# ---- pages that are kept -----------------------------------------------------------------------------------------------------------------
def test_pages_that_the_caller_keeps(pkg, torch_cuda):
    """A prefix whose counts are raised outlives its slot, is not given to another, moves with a compaction, and is free when its counts are lowered."""
    p, refs, pages, kv = pool(pkg)
    for q in (5, 6):
        refs[q] += 1
    p.put(refs)
    pkg.pages_free(p.pool, p.ints([2, 0]))
    kv[2] = kv[0] = 0
    refs = [0, 0, 1, 1, 1, 1, 1, 0, 0, 1, 0, 0, 0, 0]
    p.expect(refs, pages, kv, 0, FREE)
    pkg.pages_take(p.pool, p.ints([0, 0, 0, 0, 0, 0, 60]), p.ws)
    kv[5], pages[5] = 60, [0, 1, 7, 8]
    for q in pages[5]:
        refs[q] = 1
    p.expect(refs, pages, kv, 0, TAKE)
    pkg.pages_free(p.pool, p.ints([1]))                                               # 2, 3 and 4
    kv[1] = 0
    moved = p.ints([0] * 14)
    pkg.pages_compact(p.pool, p.cache, p.pages, p.refs, moved, p.ws)                  # 7 in use: 0 1 5 6 7 8 9, of which 7, 8, 9 go to 2, 3, 4
    assert moved.tolist() == [0, 1, -1, -1, -1, 5, 6, 2, 3, 4, -1, -1, -1, -1]
    refs, pages[5], pages[3][0] = [1] * 7 + [0] * 7, [0, 1, 2, 3], 4
    p.expect(refs, pages, kv, 0, COMPACT)
    p.moved([(7, 2, 16), (8, 3, 16), (9, 4, 16)])
    p.refs[5:7] -= 1
    pkg.pages_take(p.pool, p.ints([0, 33, 33, 33, 33, 33, 33]), p.ws)
    kv[0], pages[0], refs[7] = 33, [5, 6, 7, -7], 1
    p.expect(refs, pages, kv, 0, TAKE)


# ---- anything ------------------------------------------------------------------------------------------------------------------------------
# One block and a cluster of eight, by the pages and by the slots; lists above and below the length where children are compared in shared memory.
@pytest.mark.parametrize("num_pages,num_seqs,max_pages", [(1, 1, 1), (40, 7, 3), (300, 31, 5), (17000, 33, 9), (2000, 700, 4), (20011, 1100, 3)])
def test_numbers_of_all_kinds_stay_inside(pkg, torch_cuda, num_pages, num_seqs, max_pages):
    p = Pool(pkg, num_pages, 16, num_seqs, max_pages)
    rng = random.Random(num_pages)
    odd = [0, 1, -1, 15, 16, 17, num_pages - 1, num_pages, num_seqs - 1, num_seqs, 16 * max_pages, 16 * max_pages + 1, BIG, BIG - 1, -BIG, -BIG - 1]

    def any_ints(n, sane):
        return [rng.choice(odd) if rng.random() < 0.1 else rng.randrange(sane) for _ in range(n)]
    n = rng.randint(1, num_seqs)
    lists = [p.ints([0] * k) for k in (num_seqs + 1, n, n, num_pages)]
    out = (p.ints([0] * (num_seqs * max_pages)).view(num_seqs, max_pages), p.ints([0] * num_pages))
    for turn in range(6):
        p.put(any_ints(num_pages, 2), torch.tensor(any_ints(num_seqs * max_pages, num_pages)).view(num_seqs, max_pages).tolist(), any_ints(num_seqs, 16 * max_pages + 1))
        p.kv[:num_seqs // 2] = 0                                                      # some children that may be named
        for x, sane in zip(lists, (16 * num_seqs, num_seqs, num_seqs, num_pages)):
            x.copy_(torch.tensor(any_ints(len(x), sane), dtype=torch.int32))
        pkg.pages_take(p.pool, lists[0], p.ws)
        pkg.pages_fork(p.pool, p.cache, lists[1], lists[2], p.ws)
        pkg.pages_compact(p.pool, p.cache, *out, lists[3], p.ws)
        pkg.pages_free(p.pool, lists[1])
        pkg.pages_compact(p.pool, p.cache, p.pages, p.refs, lists[3], p.ws)
        p.margins()
        assert 0 <= p.kv.min() and p.kv.max() <= 16 * max_pages or pkg.kernel_status()[0] != 0
        pkg.kernel_status_reset()
