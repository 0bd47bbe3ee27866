"""By what position the next token of a sequence is turned, through compactions, branches and more tokens: the one behind its last key's."""
import random

import pytest
import torch

from hf2q_b200 import Hf2qError, paged
from tests.test_paged_cpu import Contents, write


@pytest.mark.parametrize("seed", range(5))
def test_the_next_turn_follows_the_last_key(seed):
    rnd = random.Random(seed)
    cache = Contents(60, 4)
    pool = paged.PagePool(cache, 3, 100)
    turns = {pool.open(): []}                              # position that each kept key was turned by
    for _ in range(300):
        what, seq = rnd.choice(["write", "write", "compact", "cut", "fork", "close"]), rnd.choice(list(turns))
        mine = turns[seq]
        if what == "write":
            n = rnd.randrange(1, 9)
            if len(mine) + n > pool.max_length or n > 4 * (pool.n_free_pages - 1):
                continue
            first = pool.length_of(seq) + pool.shift_of(seq)
            assert first == (mine[-1] + 1 if mine else 0)
            pool.reserve(seq, n)
            pool.advance(seq, n)
            mine += range(first, first + n)
        elif what == "fork" and len(turns) < 3:
            turns[pool.fork(seq)] = list(mine)
        elif what == "close" and len(turns) > 1:
            pool.close(seq)
            del turns[seq]
        elif what in ("compact", "cut") and pool.n_free_pages > len(mine) // 4 + 1:
            keep = [i for i in range(len(mine)) if i < 3 or rnd.random() < 0.7] if what == "compact" else list(range(rnd.randrange(len(mine) + 1)))
            pool.compact(seq, keep)
            turns[seq] = [mine[i] for i in keep]
        for s in range(3):
            assert int(pool.shift[s]) == (pool.shift_of(s) if s in turns else 0)


def test_first_positions_and_the_last_ones():
    pool = paged.PagePool(Contents(80, 4), 1, 300)
    s = pool.open()
    pool.reserve(s, 200)
    pool.advance(s, 200)
    pool.compact(s, [*range(4), *range(150, 200)])
    assert pool.length_of(s) == 54 and pool.length_of(s) + pool.shift_of(s) == 200
    pool.compact(s, range(54))                             # nothing more is forgotten
    assert pool.length_of(s) + pool.shift_of(s) == 200
    pool.compact(s, range(4))                              # back to the first ones
    assert pool.length_of(s) + pool.shift_of(s) == 4


def test_every_call_that_reaches_the_device_keeps_its_owners_order():
    inside, calls = [], []

    class Order:
        def __enter__(self):
            inside.append(1)

        def __exit__(self, *error):
            inside.pop()

    class Watched(Contents):
        def copy_rows(self, src, dst):
            calls.append(bool(inside))
            super().copy_rows(src, dst)

    cache = Watched(12, 4)
    pool = paged.PagePool(cache, 3, 40, Order)
    plain = pool._publish
    pool._publish = lambda seq: (calls.append(bool(inside)), plain(seq))
    a = pool.open()
    pool.reserve(a, 10)
    pool.advance(a, 10)
    b = pool.fork(a)
    pool.reserve(b, 3)                                     # copies the page that both share
    pool.advance(b, 3)
    pool.compact(b, range(1, 13, 2))
    pool.close(a)
    pool.pack()
    assert len(calls) >= 7 and all(calls) and not inside
    with pytest.raises(RuntimeError):
        pool.close(a)
    assert not inside


def full(pages, size, more=0):
    """A pool without a free page but ``more``: one sequence."""
    cache = Contents(pages + more, size)
    pool = paged.PagePool(cache, 3, (pages + more) * size)
    return cache, pool, add(cache, pool, pool.open(), pages * size)


def add(cache, pool, seq, n):
    write(cache, pool, seq, list(range(n)))
    return seq


def holds(cache, pool, seq):
    pages = pool.pages_of(seq)
    assert len(set(pages)) == len(pages) and len(pages) == -(-pool.length_of(seq) // cache.page)
    return [cache.rows[pages[i // cache.page] * cache.page + i % cache.page] for i in range(pool.length_of(seq))]


@pytest.mark.parametrize("more", [0, 1])
@pytest.mark.parametrize("keep", [range(0, 64, 4), range(60), range(1, 64), range(63), [*range(20), *range(21, 64)], [*range(32), *range(40, 64)], [63], [], range(64),
                                  [*range(16), 63]])
def test_a_full_pool_can_be_compacted(keep, more):
    cache, pool, s = full(4, 16, more)
    pool.compact(s, keep)
    assert holds(cache, pool, s) == list(keep)
    assert pool.n_free_pages == 4 + more - -(-len(keep) // 16)
    pool.compact(s, range(pool.length_of(s)))
    assert holds(cache, pool, s) == list(keep)


def test_an_end_that_is_forgotten_moves_nothing():
    """Rejected drafts: also where the pages are shared."""
    cache, pool, s = full(4, 16)
    pool.close(add(cache, pool, pool.fork(s), 0))
    b = pool.fork(s)
    cache.copy_rows = None
    pool.compact(b, range(35))
    assert holds(cache, pool, b) == list(range(35)) and pool.pages_of(b) == pool.pages_of(s)[:3] and pool.n_free_pages == 0
    pool.compact(s, range(20))
    assert holds(cache, pool, s) == list(range(20)) and pool.n_free_pages == 1


def test_shared_pages_are_not_packed_in_place():
    cache, pool, s = full(4, 16, 1)
    b = pool.fork(s)
    with pytest.raises(RuntimeError, match="no free page"):
        pool.compact(b, range(1, 64))                      # four pages of its own
    assert holds(cache, pool, b) == holds(cache, pool, s) == list(range(64))
    pool.compact(b, range(1, 64, 5))
    assert holds(cache, pool, b) == list(range(1, 64, 5)) and holds(cache, pool, s) == list(range(64)) and pool.n_free_pages == 0
    pool.compact(s, range(1, 17))                          # s has its pages for itself now, and packs in them
    assert holds(cache, pool, s) == list(range(1, 17))


@pytest.mark.parametrize("seed", range(8))
def test_compactions_of_pools_that_are_nearly_full(seed):
    rnd = random.Random(seed)
    size = rnd.choice([1, 4, 16])
    cache = Contents(rnd.randrange(6, 20), size)
    pool = paged.PagePool(cache, 3, cache.pages * size)
    want = {pool.open(): [], pool.open(): []}
    mark = 0
    for _ in range(120):
        s = rnd.choice(list(want))
        n = rnd.randrange(0, size * cache.pages)
        try:
            write(cache, pool, s, list(range(mark, mark + n)))
            want[s], mark = want[s] + list(range(mark, mark + n)), mark + n
        except (RuntimeError, Hf2qError):
            pass
        if rnd.random() < 0.2 and len(want) < 3:
            want[pool.fork(s)] = list(want[s])
        part = rnd.choice([0.3, 0.9, 0.99])
        keep = [i for i in range(len(want[s])) if rnd.random() < part]
        try:
            pool.compact(s, keep)
            want[s] = [want[s][i] for i in keep]
        except RuntimeError:
            assert any(pool._refs[p] > 1 for p in pool.pages_of(s))
        if rnd.random() < 0.1 and len(want) > 1:
            pool.close(s)
            del want[s]
        for x, values in want.items():
            assert holds(cache, pool, x)[:len(values)] == values and pool.length_of(x) == len(values)
        assert pool.n_free_pages == cache.pages - len({p for x in want for p in pool.pages_of(x)})


def test_a_sequence_does_not_pass_the_pools_longest():
    """6 positions in pages of 4: the last page has room for two that a batch of up to 6 would not take."""
    pool = paged.PagePool(Contents(4, 4), 1, 6)
    s = pool.open()
    pool.reserve(s, 6)
    with pytest.raises(Hf2qError):
        pool.advance(s, 7)
    pool.advance(s, 6)
    with pytest.raises(Hf2qError):
        pool.advance(s, 1)
    assert pool.length_of(s) == 6


def test_rows_too_far_apart_for_the_entries_are_refused():
    """A distance is passed in 32 bits."""
    class OnCpu:
        device = -1

    rows = lambda n, apart: paged._rows(torch.empty((n, apart), device="meta")[:, :64], "x", (torch.float32,), n, 64, OnCpu())
    assert rows(3, 70) == 70 and rows(3, (1 << 32) - 1) == (1 << 32) - 1
    assert rows(1, 1 << 33) == 64                          # (one row has no distance)
    with pytest.raises(Hf2qError):
        rows(3, 1 << 32)
