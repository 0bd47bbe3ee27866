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


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("longer", [1.3, 1.4, 4, 50])
@pytest.mark.parametrize("window", [0, 500])
def test_calls_laid_out_for_longer_sequences(gpu_ctx, case, longer, window):
    """Where all sequences are much shorter than the call allows, the parts are too."""
    lengths, kv, group, dim, _, _ = CASES[case]
    c = Pages(lengths, kv, group, dim, 64, torch.int8, seed=case, ld_extra=3)
    got = torch.empty((c.rows, c.heads * dim), device="cuda")
    c.cache(gpu_ctx).attend(0, c.batch(gpu_ctx, max_length=int(longer * int(c.length.max()))), c.q.cuda(), c.heads, got, window=window, sinks=5)
    gpu_ctx.check_status()
    want, tol = attention(c, c.q, torch.float32, torch.float32, window=window, sinks=5)
    close(got, want, tol)


def test_more_sequences_than_a_warp_has_lanes(gpu_ctx):
    c = Pages([(1, 60 * i) for i in range(40)], 1, 4, 64, 32, torch.int8, seed=1)
    got = torch.empty((c.rows, c.heads * 64), device="cuda")
    c.cache(gpu_ctx).attend(0, c.batch(gpu_ctx, max_length=20000), c.q.cuda(), c.heads, got)
    gpu_ctx.check_status()
    want, tol = attention(c, c.q, torch.float32, torch.float32)
    close(got, want, tol)


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


def test_calls_on_two_streams_at_once(gpu_ctx):
    """Each with a batch, and so a scratch, of its own; eager and replayed."""
    sets = []
    for seed, lengths in enumerate(([(200, 1500), (90, 300)], [(1, 6000), (1, 700)], [(130, 0)], [(40, 2600)])):
        c = Pages(lengths, 2, 4, 128, 32, torch.int8 if seed % 2 else torch.bfloat16, seed=seed)
        sets.append((c, c.cache(gpu_ctx), c.q.cuda()))
    run = lambda s, batch, out: s[1].attend(0, batch, s[2], s[0].heads, out)
    new = lambda s: torch.empty((s[0].rows, s[0].heads * 128), device="cuda")
    want = []
    for s in sets:
        want.append(new(s))
        run(s, s[0].batch(gpu_ctx), want[-1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    batches = [[s[0].batch(gpu_ctx) for s in sets] for _ in streams]
    outs = [[[new(s) for s in sets] for _ in range(6)] for _ in streams]
    torch.cuda.synchronize()
    graphs = []
    for k, st in enumerate(streams):
        with torch.cuda.stream(st):
            for s, b, o in zip(sets, batches[k], outs[k][0]):                       # (makes the scratch)
                run(s, b, o)
    torch.cuda.synchronize()
    for k, st in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            for out in outs[k][3:]:
                for i in range(len(sets)):
                    i = i if k == 0 else len(sets) - 1 - i
                    run(sets[i], batches[k][i], out[i])
        graphs.append(g)
    torch.cuda.synchronize()
    for out in (o for k in outs for o in k):
        for o in out:
            o.zero_()
    torch.cuda.synchronize()
    for r in range(3):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                for i in range(len(sets)):
                    i = i if k == 0 else len(sets) - 1 - i
                    run(sets[i], batches[k][i], outs[k][r][i])
    for k, st in enumerate(streams):
        with torch.cuda.stream(st):
            graphs[k].replay()
    torch.cuda.synchronize()
    gpu_ctx.check_status()
    assert all(torch.equal(o, w) for k in outs for out in k for o, w in zip(out, want))
