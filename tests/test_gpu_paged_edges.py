"""Calls over pages at the edges of what is allowed: no rows, rows of nobody, the smallest numbers."""
import pytest
import torch

from hf2q_b200 import paged
from tests.paged_util import Pages, attention, close

pytestmark = pytest.mark.gpu

BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("held", [0, 37, 9000])
@pytest.mark.parametrize("max_length", [0, 37, 20000])
def test_a_batch_without_rows(gpu_ctx, max_length, held, dtype):
    """A step in which no sequence has a token: empty tensors (which have no address) through the classes, and nothing happens."""
    c = Pages([(1, 99)], 2, 2, 64, 16, dtype, 1)
    cache = c.cache(gpu_ctx)
    before = cache.k.clone()
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = paged.PagedBatch(gpu_ctx, torch.zeros(3, **i32), torch.full((2,), held, **i32), torch.zeros((2, 700), **i32), rows=0, max_new=0, max_length=max_length)
    rope = paged.Rope(paged.rope_frequencies(64, 10000.0).cuda())
    x, q, out = (torch.empty((0, n * 64), device="cuda") for n in (8, 4, 4))
    assert x.data_ptr() == 0
    cache.append(0, batch, rope, x, 4, q)
    cache.attend(0, batch, q, 4, out)
    gpu_ctx.check_status()
    assert torch.equal(cache.k.view(I8), before.view(I8))


@pytest.mark.parametrize("size", [2.0 ** -119, 2.0 ** -122, 2.0 ** -126, 2.0 ** -135, 2.0 ** -149])
def test_codes_of_the_smallest_numbers(gpu_ctx, size):
    """127 / top is past the f32 range there.  A value is off by half a code, a code's own share of the scale's rounding (half of the smallest
    number, 127 times over) and roundings in 32 bits."""
    c = Pages([(30, 0)], 2, 1, 64, 16, I8, 2)
    c.x.mul_(size)
    cache, q = c.cache(gpu_ctx), torch.empty((30, 128), device="cuda")
    cache.append(0, c.batch(gpu_ctx), None, c.x.cuda(), 2, q)
    gpu_ctx.check_status()
    p = torch.arange(30)
    page, row = c.table[0, p // 16].long(), p % 16
    for t, scale, heads in ((cache.k, cache.k_scale, slice(2, 4)), (cache.v, cache.v_scale, slice(4, 6))):
        want = c.x.view(30, -1, 64)[:, heads].double()
        got = t[0].cpu()[page, :, row].double() * scale[0].cpu()[page, :, row].double()[..., None]
        unit = want.abs().amax(-1, keepdim=True) / 127
        assert bool(((got - want).abs() <= 0.501 * unit + 127 * 2.0 ** -150 + 127 * 2.0 ** -23 * unit).all())


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("lengths", [[(1, 30), (1, 5000)], [(90, 40), (5, 3)], [(70, 5000)]])
def test_rows_in_front_of_the_first_sequence_are_nobodys(gpu_ctx, lengths, dtype):
    c = Pages(lengths, 2, 4, 64, 16, dtype, 3)
    front, back, width = 3, 2, c.heads * 64
    rows = front + c.rows + back
    c.start += front
    x = torch.randn((rows, c.x.shape[1]), generator=torch.Generator().manual_seed(1))
    cache, batch, q, out = c.cache(gpu_ctx), c.batch(gpu_ctx, rows=rows), torch.full((rows, width), 7.0, device="cuda"), torch.full((rows, width), 7.0, device="cuda")
    cache.attend(0, batch, torch.cat([torch.zeros((front, width)), c.q, torch.zeros((back, width))]).cuda(), c.heads, out)
    gpu_ctx.check_status()
    c.start -= front
    want, tol = attention(c, c.q, F32, F32)
    close(out[front:-back], want, tol)
    assert bool((out[:front] == 7).all()) and bool((out[-back:] == 7).all())
    cache.append(0, batch, None, x.cuda(), c.heads, q)
    gpu_ctx.check_status()
    assert torch.equal(q[front:-back].cpu(), x[front:-back, :width]) and bool((q[:front] == 7).all()) and bool((q[-back:] == 7).all())
    p = int(c.length[0]) - 1                                          # the first sequence's last row went to its last position
    got = cache.k[0, int(c.table[0, p // 16]), :, p % 16].cpu()
    row = x[front + lengths[0][0] - 1].view(-1, 64)[c.heads:c.heads + 2]
    assert torch.equal(got, row.to(BF)) if dtype == BF else torch.equal(got, (row * (127 / row.abs().amax(-1, keepdim=True))).round().to(I8))


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("scale", [-0.09, 0.0, 2.5])
@pytest.mark.parametrize("lengths", [[(1, 300)], [(1, 6000), (1, 2)], [(90, 40), (5, 3)], [(70, 5000)]])
def test_any_scale(gpu_ctx, lengths, scale, dtype):
    """Negative: the smallest product is the largest score; zero: the mean of what is seen."""
    c = Pages(lengths, 2, 4, 128, 16, dtype, 4)
    out = torch.empty((c.rows, c.heads * 128), device="cuda")
    c.cache(gpu_ctx).attend(0, c.batch(gpu_ctx), c.q.to(BF).cuda(), c.heads, out, scale=scale)
    gpu_ctx.check_status()
    want, tol = attention(c, c.q, BF, F32, scale)
    if dtype == I8:
        # Where one score is far above the others their weights fall below the f16 normal range (2^-14), where a rounding is off by half of 2^-24.  Many
        # rows: the weight of p is p * v_scale * 16 / U, U a power of two of at most twice the largest v_scale, so that p * v_scale is off by at
        # most 2^-25 U / 16 = 2^-28 of the largest v_scale, for each position, times a code of up to 127, over a sum of at least 1.  (Few rows
        # have 256 in the place of 16.)
        tol = tol + int(c.length.max()) * 127 * c.v_scale.nan_to_num(0).max().double() * 2.0 ** -28
    close(out, want, tol)


@pytest.mark.parametrize("dtype", [BF, I8])
def test_keys_and_values_without_queries(gpu_ctx, dtype):
    c = Pages([(5, 20), (1, 0)], 3, 1, 64, 16, dtype, 5)
    cache, q = c.cache(gpu_ctx), torch.empty((6, 0), device="cuda")
    rope = paged.Rope(paged.rope_frequencies(64, 10000.0).cuda())
    cache.append(0, c.batch(gpu_ctx), rope, c.x[:, 3 * 64:].cuda(), 0, q)
    whole, q = c.cache(gpu_ctx), torch.empty((6, 3 * 64), device="cuda")
    whole.append(0, c.batch(gpu_ctx), rope, c.x.cuda(), 3, q)
    gpu_ctx.check_status()
    bits = lambda t: t.view({1: I8, 2: torch.int16, 4: torch.int32}[t.element_size()])
    for a, b in ((cache.k, whole.k), (cache.v, whole.v), (cache.k_scale, whole.k_scale), (cache.v_scale, whole.v_scale)):
        assert a is None or torch.equal(bits(a), bits(b))


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("most", [1, 40])
def test_as_many_sequences_as_a_batch_may_have(gpu_ctx, most, dtype):
    """65535 of up to 16 positions, every third without a row, the last one with ``most``."""
    seqs, g = 65535, torch.Generator().manual_seed(6)
    new = torch.tensor([1, 0, 1]).repeat(seqs // 3)
    new[-1] = most
    length = torch.maximum(torch.randint(1, 17, (seqs,), generator=g), new)
    pages = torch.randperm(seqs + 2, generator=g)
    table = torch.stack([pages[:seqs], torch.full((seqs,), seqs), torch.full((seqs,), seqs + 1)], 1)
    table[:, 1:] = pages[seqs:]
    start = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)])
    rows, k = int(start[-1]), torch.randn((1, seqs + 2, 1, 16, 64), generator=g)
    v, q = torch.randn(k.shape, generator=g), torch.randn((rows, 128), generator=g).to(BF)
    if dtype == I8:
        scale = [t.abs().amax(-1) / 127 for t in (k, v)]
        k, v = ((t / s[..., None]).round().to(I8) for t, s in zip((k, v), scale))
        cache = paged.PagedCache(gpu_ctx, *(t.cuda() for t in (k, v, *scale)))
        k, v = (t.double() * s.double()[..., None] for t, s in zip((k, v), scale))
    else:
        k, v = k.to(BF), v.to(BF)
        cache = paged.PagedCache(gpu_ctx, k.cuda(), v.cuda())
    i32 = lambda t: t.to(torch.int32).cuda()
    out = torch.empty((rows, 128), device="cuda")
    cache.attend(0, paged.PagedBatch(gpu_ctx, i32(start), i32(length), i32(table), rows=rows, max_new=most, max_length=48), q.cuda(), 2, out)
    gpu_ctx.check_status()
    seq = torch.repeat_interleave(torch.arange(seqs), new)
    pos = length[seq] - start[seq + 1] + torch.arange(rows)
    k, v = (t[0, table].reshape(seqs, 48, 64).double()[seq] for t in (k, v))
    x = torch.einsum("rhd,rjd->rhj", q.double().view(rows, 2, 64), k) / 8
    x = x.masked_fill((torch.arange(48)[None] > pos[:, None])[:, None], float("-inf"))
    p = torch.softmax(x, -1)
    want, spread = torch.einsum("rhj,rjd->rhd", p, v), torch.einsum("rhj,rjd->rhd", p, v.abs())
    # weights rounded to 16 bits, scores of exact products summed in 32: a weight is off by 2^-8 and a few 2^-16 at most
    assert bool(((out.cpu().double().view(rows, 2, 64) - want).abs() <= spread * (2.0 ** -8 + 2.0 ** -12)).all())
