"""Attention over a paged cache whose positions are split: few and many parts, sequences that have none in most of them, every result type."""
import pytest
import torch

from tests.paged_util import Pages, attention, close

pytestmark = pytest.mark.gpu


def parts_of(batch, cache, heads):
    return batch.scratch(cache.structs[0], heads, 0, 0).numel() // (batch.rows * heads * (cache.dim + 2) * 4)


# (new, before) of the sequences, KV heads, group, dim, at least and at most so many parts
CASES = [
    ([(1, 700)], 1, 4, 128, 2, 16), ([(1, 5000)], 1, 3, 64, 17, 60), ([(1, 9000), (1, 3), (1, 0), (1, 2500)], 2, 4, 128, 17, 80), ([(2, 6000), (1, 1)], 1, 8, 64, 17, 60),
    ([(40, 3000)], 1, 2, 128, 2, 16), ([(33, 9000)], 1, 4, 64, 17, 40), ([(70, 9100), (3, 90), (41, 0)], 1, 4, 128, 17, 40), ([(300, 2500)], 2, 3, 64, 2, 16),
]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_parts_join_to_the_whole(gpu_ctx, case, dtype, out):
    lengths, kv, group, dim, least, most = CASES[case]
    c = Pages(lengths, kv, group, dim, 32, dtype, seed=case)
    cache, batch = c.cache(gpu_ctx), c.batch(gpu_ctx)
    assert least <= parts_of(batch, cache, c.heads) <= most
    got = torch.full((c.rows, c.heads * dim + 3), 5.0, dtype=out, device="cuda")                   # rows that lie apart, between two 16-byte boundaries
    cache.attend(0, batch, c.q.cuda(), c.heads, got)
    gpu_ctx.check_status()
    want, tol = attention(c, c.q, torch.float32, out)
    close(got[:, :c.heads * dim], want, tol)
    assert bool((got[:, c.heads * dim:] == 5).all())


def test_parts_give_the_same_sums_every_time(gpu_ctx):
    for lengths in ([(1, 9000), (1, 2500)], [(70, 9100)]):
        c = Pages(lengths, 2, 4, 128, 16, torch.int8, seed=3)
        cache, batch, q = c.cache(gpu_ctx), c.batch(gpu_ctx), c.q.cuda()
        got = [torch.empty((c.rows, c.heads * 128), device="cuda") for _ in range(4)]
        for g in got:
            batch.scratch(cache.structs[0], c.heads, 0, 0).fill_(255)                              # (NaN: nothing is read that this call has not written)
            cache.attend(0, batch, q, c.heads, g)
        gpu_ctx.check_status()
        assert all(torch.equal(g, got[0]) for g in got) and not bool(got[0].isnan().any())
