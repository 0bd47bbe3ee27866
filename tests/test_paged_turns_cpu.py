"""By what position the next token of a sequence is turned, through compactions, branches and more tokens: the one behind its last key's."""
import random

import pytest

from hf2q_b200 import paged
from tests.test_paged_cpu import Contents


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
