"""The pages of a cache, taken, forked, freed, compacted and copied: whole numbers and bytes, so everything has to be equal to the lists' (pages_helpers.py)."""
import random

import pytest
import torch

from pages_helpers import Device, Model, equal_bits, moved_bits

pytestmark = pytest.mark.gpu


def pair(pkg, num_pages, page, num_seqs, max_pages, **kw):
    pkg.kernel_status_reset()
    m, d = Model(num_pages, page, num_seqs, max_pages), Device(pkg, num_pages, page, num_seqs, max_pages, **kw)
    d.load(m)
    return m, d


def scatter(m, rng, lengths, shared=0.3):
    """Slots of these lengths on random pages, some of the full ones in common with the slot before."""
    order = list(range(len(m.refs)))
    rng.shuffle(order)
    for b, n in enumerate(lengths):
        m.kv[b] = n
        for e in range(m.held(b)):
            full = (e + 1) * m.page <= n
            if b and full and e < m.held(b - 1) and (e + 1) * m.page <= m.kv[b - 1] and rng.random() < shared:
                m.pages[b][e] = m.pages[b - 1][e]
                m.refs[m.pages[b][e]] += 1
            else:
                m.pages[b][e] = order.pop()
                m.refs[m.pages[b][e]] = 1


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("bits,gap", [(16, 0), (8, 0), (16, 48), (8, 48)])
def test_a_server_s_life(pkg, torch_cuda, page, bits, gap):
    """Takes, forks, frees and compactions in turn, the pool full at times."""
    S, W, N = 23, 9, 70
    m, d = pair(pkg, N, page, S, W, bits=bits, gap=gap, d=16 if page > 64 else 32, seed=page)
    rng = random.Random(page + bits)
    for step in range(60):
        op = rng.choice(["take", "take", "fork", "free", "compact"])
        if op == "take":
            new = [min(rng.choice([0, 1, 1, page - 1, page, 2 * page + 3]), W * page - n) if rng.random() < 0.4 else 0 for n in m.kv]
            m.take(new)
            pkg.pages_take(d.pool, d.starts(new, rng.randint(0, 5)), d.ws)
        elif op == "fork":
            empty = [b for b in range(S) if m.kv[b] == 0]
            rng.shuffle(empty)
            children = empty[:rng.randint(0, len(empty))]
            parents = [rng.randrange(S) for _ in children]
            before = d.bits()
            moves = m.fork(parents, children)
            pkg.pages_fork(d.pool, d.cache, d.ints(*parents), d.ints(*children), d.ws)
            assert equal_bits(d.bits(), moved_bits(before, moves)), step
        elif op == "free":
            seqs = [b for b in range(S) if rng.random() < 0.3] + [rng.randrange(S)] * 2
            m.free(seqs)
            pkg.pages_free(d.pool, d.ints(*seqs))
        else:
            before = d.bits()
            m.pages, m.refs, moved, pairs = m.compact()
            got = d.ints(*[5] * N)
            pkg.pages_compact(d.pool, d.cache, d.pages, d.refs, got, d.ws)
            assert got.tolist() == moved
            assert equal_bits(d.bits(), moved_bits(before, [(p, q, page) for p, q in pairs])), step
        d.same(m)
        assert (pkg.kernel_status()[0] != 0) == m.wrong
        if m.wrong:
            m.wrong = False
            pkg.kernel_status_reset()


# Pools below, at and above a block's thousand threads, eight segments, several tiles of a segment.
@pytest.mark.parametrize("num_pages", [1, 2, 7, 8, 9, 1000, 1024, 8191, 8192, 8193, 20000, 100003])
def test_pools_of_all_sizes(pkg, torch_cuda, num_pages):
    S, W = 41, max(1, min(3000, num_pages // 20))
    m, d = pair(pkg, num_pages, 16, S, W, H=1, seed=1)
    rng = random.Random(num_pages)
    scatter(m, rng, [min(rng.randint(0, 16 * W), 16 * max(0, num_pages // 60)) for _ in range(20)] + [0] * 21)
    d.load(m)
    new = [0] * 20 + [rng.randint(0, 16 * W // 2) for _ in range(21)]
    m.take(new)
    pkg.pages_take(d.pool, d.starts(new), d.ws)
    d.same(m)
    gone = [b for b in range(S) if b % 3 == 0]
    m.free(gone)
    pkg.pages_free(d.pool, d.ints(*gone))
    d.same(m)
    before = d.bits()
    pages, refs, moved, pairs = m.compact()
    po, ro, mo = torch.full_like(d.pages, -9), torch.full_like(d.refs, -9), torch.full_like(d.refs, -9)
    pkg.pages_compact(d.pool, d.cache, po, ro, mo, d.ws)                     # into arrays of its own
    d.same(m)                                                               # the pool's stay
    assert ro.tolist() == refs and mo.tolist() == moved
    for b in range(S):
        assert po[b].tolist() == pages[b][:m.held(b)] + [-9] * (W - m.held(b))
    assert equal_bits(d.bits(), moved_bits(before, [(p, q, 16) for p, q in pairs]))


@pytest.mark.parametrize("num_seqs", [1, 31, 1023, 1025, 8200, 20000])
def test_many_slots(pkg, torch_cuda, num_seqs):
    m, d = pair(pkg, 2 * num_seqs + 40, 16, num_seqs, 3, H=1)
    rng = random.Random(num_seqs)
    new = [rng.choice([0, 1, 16, 17, 40]) for _ in range(num_seqs)]
    m_free = 2 * num_seqs + 40
    rank = 0                                                                # the lists' search for a free page would take long
    for b, n in enumerate(new):
        for e in range(-(-n // 16)):
            m.pages[b][e] = rank if rank < m_free else -1
            if rank < m_free:
                m.refs[rank] = 1
            rank += 1
        m.kv[b] = n
    pkg.pages_take(d.pool, d.starts(new), d.ws)
    d.same(m)
    assert (pkg.kernel_status()[0] == 4) == (rank > m_free)
    order = list(range(num_seqs))
    rng.shuffle(order)
    m.free(order)
    pkg.pages_free(d.pool, d.ints(*order))
    d.same(m)
    assert not any(m.refs)


def test_many_forks(pkg, torch_cuda):
    """More entries than a block has threads; children without end of one parent."""
    S = 9000
    m, d = pair(pkg, 9100, 16, S, 4, H=1, bits=8)
    m.take([40, 32, 1] + [0] * (S - 3))
    children = list(range(S - 1, 2, -1))
    parents = [c % 3 for c in children]
    pages, free = [list(r) for r in m.pages[:3]], 6
    assert pages[0][:3] == [0, 1, 2] and pages[1][:2] == [3, 4] and pages[2][0] == 5
    moves = []
    for p, c in zip(parents, children):
        m.kv[c] = m.kv[p]
        for e in range(m.kv[p] // 16):
            m.pages[c][e] = pages[p][e]
            m.refs[pages[p][e]] += 1
        if m.kv[p] % 16:
            e = m.kv[p] // 16
            m.pages[c][e], m.refs[free] = free, 1
            moves.append((pages[p][e], free, m.kv[p] % 16))
            free += 1
    pkg.pages_take(d.pool, d.starts([40, 32, 1] + [0] * (S - 3)), d.ws)
    before = d.bits()
    pkg.pages_fork(d.pool, d.cache, d.ints(*parents), d.ints(*children), d.ws)
    d.same(m)
    got = d.bits()
    src, dst, keys = (torch.tensor(x).cuda() for x in zip(*moves))
    there = torch.arange(16, device="cuda") < keys[:, None]
    for x, y in zip(got, before):
        want = y.clone()
        want[dst] = torch.where(there.reshape(len(keys), 1, 16, *[1] * (y.dim() - 3)), y[src], y[dst])
        assert torch.equal(x, want)
    assert pkg.kernel_status()[0] == 0


def test_a_pool_without_enough_pages(pkg, torch_cuda):
    """Slots in order get what there is; the entries of the others are -1, and everything goes on from there."""
    m, d = pair(pkg, 5, 16, 4, 4)
    new = [20, 40, 33, 1]
    m.take(new)
    pkg.pages_take(d.pool, d.starts(new), d.ws)
    d.same(m)
    assert m.pages[1] == [2, 3, 4, -7] and m.pages[2] == [-1, -1, -1, -7] and m.pages[3][0] == -1
    assert pkg.kernel_status()[0] == 4 and pkg.kernel_status()[2] == 60
    pkg.kernel_status_reset()
    m.free([3])
    pkg.pages_free(d.pool, d.ints(3))
    d.same(m)
    assert pkg.kernel_status()[0] == 0                                      # -1 is nobody's page
    moves = m.fork([0, 2], [3, 3])                                          # no page for the child's last keys; the second entry names it again
    before = d.bits()
    pkg.pages_fork(d.pool, d.cache, d.ints(0, 2), d.ints(3, 3), d.ws)
    d.same(m)
    assert moves == [] and m.pages[3][:2] == [0, -1] and m.refs[0] == 2 and equal_bits(before, d.bits())
    assert pkg.kernel_status()[0] in (4, 5) and pkg.kernel_status()[2] == 61
    m.free([0, 1, 2, 3])
    pkg.pages_free(d.pool, d.ints(0, 1, 2, 3))
    d.same(m)
    assert m.refs == [0] * 5


@pytest.mark.parametrize("parents,children", [([0, 1], [3, 3]), ([0], [1]), ([0], [0]), ([2], [2]), ([0, 0], [-1, 3]), ([5, 0], [3, 2]), ([-3], [3]), ([2, 0], [3, 2]), ([0, 2], [2, 3])])
def test_forks_that_name_slots_wrongly(pkg, torch_cuda, parents, children):
    """The same child twice, a child with keys, its own parent, slots that there are not: those entries change nothing. An empty slot's copy is empty."""
    m, d = pair(pkg, 30, 16, 4, 4)
    new = [20, 40, 0, 0]
    m.take(new)
    pkg.pages_take(d.pool, d.starts(new), d.ws)
    before = d.bits()
    moves = m.fork(parents, children)
    pkg.pages_fork(d.pool, d.cache, d.ints(*parents), d.ints(*children), d.ws)
    d.same(m)
    assert equal_bits(d.bits(), moved_bits(before, moves))
    assert (pkg.kernel_status()[0] == 5) == m.wrong


def test_wrong_lengths_and_pages_stay_inside(pkg, torch_cuda):
    big = 2 ** 31 - 1
    m, d = pair(pkg, 40, 16, 6, 4)
    new = [20, 40, 64, 5, 0, 0]
    m.take(new)
    pkg.pages_take(d.pool, d.starts(new), d.ws)
    d.kv[1], d.kv[2], d.pages[0, 0], d.pages[3, 0] = big, -big - 1, 40, -big
    guard = [x.clone() for x in (d.refs, d.pages, d.kv)]
    for call in (lambda: pkg.pages_take(d.pool, d.ints(0, big, -big, big, 0, -5, big), d.ws), lambda: pkg.pages_fork(d.pool, d.cache, d.ints(0, 1), d.ints(4, 5), d.ws),
                 lambda: pkg.pages_compact(d.pool, d.cache, d.pages, d.refs, d.ints(*[0] * 40), d.ws), lambda: pkg.pages_free(d.pool, d.ints(0, 1, 2, 3, 4, 5, 6, -1, big))):
        pkg.kernel_status_reset()
        for x, y in zip((d.refs, d.pages, d.kv), guard):
            x.copy_(y)
        call()
        torch.cuda.synchronize()
        assert pkg.kernel_status()[0] in (2, 3, 4, 5)
        assert d.pages.min() >= -big and d.refs.min() >= 0
    pkg.kernel_status_reset()


def test_a_page_freed_too_often_stays_free(pkg, torch_cuda):
    m, d = pair(pkg, 10, 16, 3, 4)
    d.kv[0], d.kv[1] = 32, 16
    d.pages[0, 0], d.pages[0, 1], d.pages[1, 0] = 4, 5, 4                   # page 4 is named twice and counted once
    d.refs[4], d.refs[5] = 1, 1
    pkg.pages_free(d.pool, d.ints(0, 1))
    torch.cuda.synchronize()
    assert d.refs.tolist() == [0] * 10 and pkg.kernel_status()[0] == 2 and pkg.kernel_status()[2] == 62


@pytest.mark.parametrize("H,d_h,page,bits,gap", [(1, 16, 16, 8, 0), (1, 16, 16, 16, 0), (8, 128, 256, 16, 0), (3, 64, 32, 8, 16), (16, 128, 128, 8, 0), (5, 32, 16, 16, 160), (40, 128, 256, 8, 0)])
def test_copies(pkg, torch_cuda, H, d_h, page, bits, gap):
    d = Device(pkg, 33, page, 1, 1, H=H, d=d_h, bits=bits, gap=gap, seed=H)
    pkg.kernel_status_reset()
    rng = random.Random(H)
    order = list(range(33))
    rng.shuffle(order)
    for n in (0, 1, 13):
        before = d.bits()
        src, dst = [order[rng.randrange(13)] for _ in range(n)], order[20:20 + n]
        pkg.pages_copy(d.cache, d.ints(*src), d.ints(*dst))
        torch.cuda.synchronize()
        assert equal_bits(d.bits(), moved_bits(before, [(p, q, page) for p, q in zip(src, dst)]))
    assert pkg.kernel_status()[0] == 0
    before = d.bits()
    pkg.pages_copy(d.cache, d.ints(order[0], 33, -1, order[1]), d.ints(33, order[2], order[3], order[25]))
    torch.cuda.synchronize()
    assert equal_bits(d.bits(), moved_bits(before, [(order[1], order[25], page)]))
    assert pkg.kernel_status()[0] == 2 and pkg.kernel_status()[2] == 64


def test_gaps_between_pages_stay(pkg, torch_cuda):
    d = Device(pkg, 9, 16, 1, 1, H=3, d=32, gap=32)
    whole = [x.as_strided((9, 3 * 16 * 32 + 32), (3 * 16 * 32 + 32, 1)) for x in d.parts]
    for x in whole:
        x[:, -32:] = 5
    pkg.pages_copy(d.cache, d.ints(1, 2), d.ints(3, 4))
    torch.cuda.synchronize()
    assert all(torch.all(x[:, -32:] == 5) for x in whole)


def test_a_captured_step_follows_the_arrays(pkg, torch_cuda):
    """Take, fork, free and compact in one graph, on another stream, replayed over changed lists."""
    m, d = pair(pkg, 300, 16, 12, 8, bits=8)
    starts, parents, children, gone, moved = d.starts([0] * 12), d.ints(0, 0), d.ints(0, 0), d.ints(0, 0), d.ints(*[0] * 300)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            pkg.pages_take(d.pool, starts, d.ws, stream=side)
            pkg.pages_fork(d.pool, d.cache, parents, children, d.ws, stream=side)
            pkg.pages_free(d.pool, gone, stream=side)
            pkg.pages_compact(d.pool, d.cache, d.pages, d.refs, moved, d.ws, stream=side)
    rng = random.Random(3)
    d.load(m)
    for _ in range(25):
        new = [min(rng.choice([0, 1, 17, 40]), 128 - n) if rng.random() < 0.5 else 0 for n in m.kv]
        empty = [b for b in range(12) if m.kv[b] + new[b] == 0][:2]
        kids = empty + [-1] * (2 - len(empty))
        mothers, leave = [rng.randrange(12), rng.randrange(12)], [rng.randrange(12), rng.randrange(12)]
        for x, y in ((starts, d.starts(new)), (parents, d.ints(*mothers)), (children, d.ints(*kids)), (gone, d.ints(*leave))):
            x.copy_(y)
        before = d.bits()
        graph.replay()
        m.take(new)
        data = moved_bits(before, m.fork(mothers, kids))
        m.free(leave)
        m.pages, m.refs, want, pairs = m.compact()
        d.same(m)
        assert moved.tolist() == want
        assert equal_bits(d.bits(), moved_bits(data, [(p, q, 16) for p, q in pairs]))


def test_empty_calls(pkg, torch_cuda):
    m, d = pair(pkg, 10, 16, 3, 4)
    none = d.ints()
    pkg.pages_take(d.pool, d.starts([0, 0, 0]), d.ws)
    pkg.pages_fork(d.pool, d.cache, none, none, d.ws)
    pkg.pages_free(d.pool, none)
    pkg.pages_copy(d.cache, none, none)
    moved = d.ints(*[3] * 10)
    pkg.pages_compact(d.pool, d.cache, d.pages, d.refs, moved, d.ws)
    d.same(m)
    assert moved.tolist() == [-1] * 10 and pkg.kernel_status()[0] == 0
    with pytest.raises(pkg.EfaError, match="memory of the host"):
        pkg.pages_free(d.pool, torch.zeros(1, dtype=torch.int32))
