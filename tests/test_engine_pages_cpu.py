"""The engine over a decoder whose sequences share a pool: who is admitted together, and what is left when a call fails."""
import pytest
import torch

from hf2q_b200 import paged
from hf2q_b200.engine import Engine
from tests.test_paged_cpu import Contents


class Pooled:
    """Continues a sequence with the sum of its tokens so far, then one more each time; its places are taken from a real pool."""

    def __init__(self, pages, n_slots, size=4):
        self.n_slots, self.pool, self.size = n_slots, paged.PagePool(Contents(pages, size), n_slots, 1000), size
        self.sums, self.tok, self.most, self.fail = {}, torch.zeros(1), 0, None

    def fits(self, lengths):
        return sum(-(-n // self.size) for n in lengths) <= self.pool.n_free_pages

    def open_slot(self):
        slot = self.pool.open()
        self.sums[slot] = 0
        return slot

    def close_slot(self, slot):
        self.pool.close(slot)
        del self.sums[slot]

    def bind(self, slot):
        self.slot, self.tok = slot, torch.tensor([self.sums[slot]])

    def _grow(self, slot, n):
        self.pool.reserve(slot, n)
        self.pool.advance(slot, n)
        self.most = max(self.most, len(self.sums))

    def extend(self, slot, ids, want):
        if self.fail in ids.tolist():
            raise ValueError("a call fails")
        self._grow(slot, ids.numel())
        self.sums[slot] += int(ids.sum())

    def generate(self, n):
        self._grow(self.slot, n)
        return torch.arange(n) + self.sums[self.slot] + 1


def want(prompts, n_new):
    return [list(range(sum(p), sum(p) + n_new)) for p in prompts]


@pytest.mark.parametrize("pages,together", [(4, 1), (7, 1), (8, 2), (11, 2), (12, 3), (40, 3)])
def test_prompts_wait_for_pages(pages, together):
    """Each takes 10 tokens and 6 more but one: 15 places, four pages."""
    m = Pooled(pages, 3)
    prompts = [[i] * 10 for i in range(5)]
    assert Engine(m).generate(prompts, 6) == want(prompts, 6)
    assert m.most == together and m.pool.n_free_pages == pages


def test_a_prompt_that_never_fits_is_refused_before_anything_runs():
    m = Pooled(4, 2)
    with pytest.raises(RuntimeError, match="prompt 1"):
        Engine(m).generate([[1, 2], [3] * 12], 6)          # 17 places
    assert m.most == 0 and m.pool.n_free_pages == 4
    assert Engine(m).generate([[1, 2], [3] * 11], 6) == want([[1, 2], [3] * 11], 6)


def test_slots_are_given_back_when_a_call_fails():
    m = Pooled(20, 3)
    m.fail = 9
    with pytest.raises(ValueError):
        Engine(m).generate([[1], [2], [9], [3]], 4)
    assert m.pool.n_free_pages == 20 and not m.sums
    m.fail = None
    assert Engine(m).generate([[1], [2], [9], [3]], 4) == want([[1], [2], [9], [3]], 4)
