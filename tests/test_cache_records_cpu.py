"""CPU checks of the cache's records: shared pages, compaction, and what the copies refuse."""
import array
import ctypes
import random

import pytest
import torch


def _pool(n_pages=20, batch=4, max_pages=8, page=16):
    from treeattn_b200.paged import PagePool
    return PagePool(n_pages, batch, max_pages, page, device='cpu')


def _consistent(pool):
    """Each page is free or held by as many sequences as refs says, and the table names what the sequences hold."""
    count = [0] * pool.n_pages
    for own in pool.owned:
        assert len(set(own)) == len(own)
        for p in own:
            count[p] += 1
    assert count == pool.refs
    assert sorted(pool.free) == [p for p in range(pool.n_pages) if not count[p]]
    for b, own in enumerate(pool.owned):
        assert pool.table[b, :len(own)].tolist() == own


def test_fork_shares_full_pages():
    pool = _pool()
    pool.reserve([40, 20, 0, 16])
    held = [list(o) for o in pool.owned]
    pool.fork([0, 0, 1], [2, 1, 0], [40, 40, 20])  # 0 is a source and a destination, and so is 1
    assert pool.owned == [held[1][:1], held[0][:2], held[0][:2], held[3]]
    assert pool.refs[held[0][0]] == 2 and held[0][2] in pool.free and held[1][1] in pool.free
    _consistent(pool)
    pool.fork([3, 2], [3, 0], [16, 33])  # a sequence onto itself keeps what it has
    assert pool.owned[3] == held[3] and pool.owned[0] == held[0][:2]
    _consistent(pool)


def test_shared_pages_are_replaced_before_they_are_written():
    pool = _pool()
    pool.reserve([64, 0, 0, 0])
    pool.fork([0, 0], [1, 2], [64, 64])
    pool.reserve([70, 70, 70, 0], [64, 64, 64, 0])
    first = [list(o) for o in pool.owned]
    assert first[0][:4] == first[1][:4] == first[2][:4] and len({o[4] for o in first[:3]}) == 3
    _consistent(pool)
    # two of them go back into page 3 and will write it again: both get one of their own, the third keeps what it reads
    pool.reserve([70, 64, 64, 0], [70, 50, 49, 0])
    assert pool.owned[0] == first[0] and len({o[3] for o in pool.owned[:3]}) == 3
    assert pool.owned[1][4] == first[1][4]
    _consistent(pool)
    # the last holder keeps a page
    pool.release(0)
    pool.reserve([0, 64, 64, 0], [0, 50, 49, 0])
    _consistent(pool)
    pool.release(1)
    pool.release(2)
    assert len(pool.free) == 20 and pool.refs == [0] * 20


def test_reserve_counts_replaced_pages():
    pool = _pool(n_pages=5)
    pool.reserve([64, 0, 0, 0])
    pool.fork([0], [1], [64])
    before = [list(o) for o in pool.owned], list(pool.free), list(pool.refs), pool.table.clone()
    with pytest.raises(MemoryError, match='2 pages wanted, 1 free'):
        pool.reserve([64, 80, 0, 0], [64, 48, 0, 0])
    assert before[:3] == (pool.owned, pool.free, pool.refs) and torch.equal(before[3], pool.table)


def test_positions_as_tensors():
    """Sequences and lengths may be tensors or arrays of whole numbers."""
    pool = _pool()
    pool.reserve(torch.tensor([40, 20, 0, 16]), torch.tensor([0, 0, 0, 0]))
    with pytest.raises(ValueError, match='once'):
        pool.fork(torch.tensor([0, 0]), torch.tensor([2, 2]), torch.tensor([40, 40]))
    pool.fork(torch.tensor([0]), torch.tensor([2]), torch.tensor([40]))
    assert pool.owned[2] == pool.owned[0][:2]
    _consistent(pool)


def test_refused_forks():
    pool = _pool()
    pool.reserve([40, 0, 0, 0])
    before = [list(o) for o in pool.owned], list(pool.refs)
    for src, dst, n, what in (([0], [4], [40], 'sequences'), ([-1], [1], [40], 'sequences'), ([0, 0], [1, 1], [40, 40], 'once'),
                              ([0], [1, 2], [40], '1 sources'), ([0], [1], [64], 'does not hold'), ([0], [1], [-1], 'does not hold')):
        with pytest.raises(ValueError, match=what):
            pool.fork(src, dst, n)
    assert before == (pool.owned, pool.refs)


def test_compact():
    pool = _pool()
    pool.reserve([40, 64, 17, 100])
    pool.fork([1], [0], [64])
    pool.release(3)
    held = [list(o) for o in pool.owned]
    with pytest.raises(MemoryError, match='held'):
        pool.compact(5)
    src, dst = pool.compact(6)
    assert pool.n_pages == 6 and all(p >= 6 for p in src) and all(p < 6 for p in dst)
    to = dict(zip(src, dst))
    assert [[to.get(p, p) for p in o] for o in held] == pool.owned
    _consistent(pool)
    assert pool.compact() == ([], []) and pool.free == []
    assert int(pool.table.max()) < 6  # unused places too
    for b in range(3):
        pool.release(b)
    pool.compact()
    assert pool.n_pages == 1 and pool.free == [0]


def test_random_use_of_a_pool():
    """Random forks, cuts, growth, compaction: never a page in two hands that one of them may write."""
    rng = random.Random(3)
    pool = _pool(n_pages=60, batch=6, max_pages=10, page=16)
    pos = [0] * 6
    for step in range(400):
        act = rng.random()
        if act < 0.45:
            new = [min(160, p + rng.randint(0, 20)) for p in pos]
            try:
                pool.reserve(new, pos)
            except MemoryError:
                b = rng.randrange(6)
                pool.release(b)
                pos[b] = 0
                continue
            for b, (p, n) in enumerate(zip(pos, new)):  # pages that get written
                for j in range(p // 16, -(-n // 16)):
                    if n > p:
                        assert pool.refs[pool.owned[b][j]] == 1
            pos = new
        elif act < 0.7:
            k = rng.randint(1, 5)
            dst, src = rng.sample(range(6), k), [rng.randrange(6) for _ in range(k)]
            pool.fork(src, dst, [pos[s] for s in src])
            was = list(pos)
            for s, d in zip(src, dst):
                pos[d] = was[s]
        elif act < 0.9:
            pos = [max(0, p - rng.randint(0, 17)) for p in pos]
        elif act < 0.95 or pool.n_pages < 45:
            b = rng.randrange(6)
            pool.release(b)
            pos[b] = 0
        else:
            held = pool.n_pages - len(pool.free)
            pool.compact(max(held, pool.n_pages - 1, 1))
        _consistent(pool)


def test_rejected_copies_without_gpu():
    """The entry point refuses bad moves with a message before any CUDA call."""
    from treeattn_b200 import _lib
    lib = _lib.load()
    a = 1 << 20

    def copy(src=(0,), dst=(1,), bufs=(a, a + 4096), size=64, n=8):
        s, d = array.array('i', src), array.array('i', dst)
        p = (ctypes.c_void_p * len(bufs))(*bufs)
        return lib.ta_record_copy(p, len(bufs), size, n, s.buffer_info()[0], d.buffer_info()[0], len(s), None)

    ring = list(range(2048))
    for kw, what in ((dict(src=(8,)), 'from record 8'), (dict(src=(-1,)), 'from record -1'), (dict(dst=(8,)), 'to 8 of 8'),
                     (dict(src=(0, 1), dst=(2, 2)), 'record 2 is written twice'), (dict(size=40), 'multiple of 16'),
                     (dict(size=0), 'bad sizes'), (dict(n=-1), 'bad sizes'), (dict(bufs=(a, None)), 'null'),
                     (dict(bufs=(a, a + 8)), 'aligned'), (dict(bufs=(a, a + 256)), 'overlap'), (dict(bufs=(a, a)), 'overlap'),
                     (dict(src=ring, dst=ring[1:] + [0], n=4000, bufs=(a,)), 'cycle of 2048'),
                     (dict(src=(0, 70000), dst=(69999, 69999), n=80000, bufs=(a,)), 'written twice')):
        assert copy(**kw) == _lib.TA_ERR_ARG
        assert 'ta_record_copy' in _lib.last_error() and what in _lib.last_error(), (kw, _lib.last_error())
    assert copy(src=(), dst=()) == _lib.TA_OK and copy(bufs=()) == _lib.TA_OK
    assert copy(src=(3, 4), dst=(3, 4)) == _lib.TA_OK  # nothing to move


def test_refused_lists():
    from treeattn_b200 import paged

    class Cache:
        def __init__(self, shape=(9, 2, 1040)):
            self.pool = torch.zeros(shape, dtype=torch.uint8)
            self.tail = torch.zeros(3, 2, 2, 2, 512, dtype=torch.bfloat16)

    one = [Cache()]
    for caches, src, dst, what in (([], [0], [1], 'no caches'), ([Cache(), Cache((8, 2, 1040))], [0], [1], 'alike'),
                                   (one, [0], [1, 2], '1 sources'), (one, [0.5], [1], 'whole numbers'),
                                   (one, [1 << 40], [1], 'whole numbers'), (one, [0], [1], 'CUDA')):
        with pytest.raises(ValueError, match='paged_copy.*' + what):
            paged.paged_copy(caches, src, dst)
    with pytest.raises(ValueError, match='paged_fork.*CUDA'):
        paged.paged_fork(one, [0], [1])


def test_reserve_looks_at_pages_only_where_some_are_shared():
    """A decode step of sequences that share nothing does not walk their pages; the count of further holders is right after every
    fork, cut, replacement, release and compaction."""
    class Pages(list):
        walked = 0

        def __getitem__(self, j):
            Pages.walked += 1
            return list.__getitem__(self, j)

    pool = _pool(n_pages=60, batch=6, max_pages=10)
    pool.reserve([100] * 6, [0] * 6)
    pool.owned = [Pages(o) for o in pool.owned]
    pool.reserve([101] * 6, [40] * 6)
    assert Pages.walked == 0
    pool.fork([0], [1], [100])
    pool.reserve([101] * 6, [40] * 6)
    assert Pages.walked > 0
    extra = lambda: sum(max(r - 1, 0) for r in pool.refs)
    assert pool.extra == extra()
    rng = random.Random(11)
    pos, some = [101] * 6, 0
    for _ in range(300):
        act = rng.random()
        if act < 0.4:
            new = [min(160, p + rng.randint(0, 20)) for p in pos]
            try:
                pool.reserve(new, pos)
                pos = new
            except MemoryError:
                pass
        elif act < 0.7:
            k = rng.randint(1, 5)
            dst, src = rng.sample(range(6), k), [rng.randrange(6) for _ in range(k)]
            pool.fork(src, dst, [pos[s] for s in src])
            was = list(pos)
            for s, d in zip(src, dst):
                pos[d] = was[s]
        elif act < 0.85:
            pos = [max(0, p - rng.randint(0, 40)) for p in pos]
        elif act < 0.95 or pool.n_pages < 45:
            b = rng.randrange(6)
            pool.release(b)
            pos[b] = 0
        else:
            pool.compact(max(pool.n_pages - len(pool.free), pool.n_pages - 1, 1))
        assert pool.extra == extra()
        some += pool.extra > 0
        _consistent(pool)
    assert some > 50
    for b in range(6):
        pool.release(b)
    assert pool.extra == 0
