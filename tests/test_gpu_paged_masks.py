"""Paged attention where something infinite or NaN lies in places that a row does not see, or does; rows that see nothing; pools past
32-bit offsets; captured calls; batches that do not fit."""
import math

import pytest
import torch

from hf2q_b200 import Hf2qError, paged
from paged_util import Pages, attention, close, turned

pytestmark = pytest.mark.gpu

BF, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def run(ctx, c, window=0, sinks=0, out_dtype=F32, **bounds):
    out = torch.full((c.rows, c.heads * c.dim), 77.0, dtype=out_dtype, device="cuda")
    c.cache(ctx).attend(0, c.batch(ctx, **bounds), c.q.to(BF).cuda(), c.heads, out, window=window, sinks=sinks)
    return out


def at(c, s, p):
    return (0, int(c.table[s, p // c.page]), slice(None), p % c.page)


# new rows a sequence: single rows, a tile of few rows, and the products of many rows with one and with two tiles
@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("where", ["k", "v", "both"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new,group,window,sinks", [(5, 3, 0, 0), (40, 4, 0, 0), (150, 2, 0, 0), (6, 2, 30, 2), (100, 4, 50, 3)])
def test_what_a_row_does_not_see_has_no_part_in_it(gpu_ctx, new, group, window, sinks, value, where, dtype):
    c = Pages([(new, 90), (3, 0)], 2, group, 64, 16, dtype, new)
    total = 90 + new
    hidden_from = 90 + new // 2                                      # seen from here on
    places = [total - 1] + ([90 - window + 3] if window else [hidden_from])      # windowed: the first rows see it, the others do not any more
    clean = Pages([(new, 90), (3, 0)], 2, group, 64, 16, dtype, new)
    for p in places:
        for name in "kv":
            if where not in (name, "both"):
                continue
            for pages, v in ((c, value), (clean, 0.0)):
                if dtype == I8:
                    getattr(pages, name + "_scale")[at(c, 0, p)] = v
                else:
                    getattr(pages, name)[at(c, 0, p)] = v
    got = run(gpu_ctx, c, window, sinks).cpu().double()
    gpu_ctx.check_status()
    want, tol = attention(clean, c.q, BF, F32, None, window, sinks)
    i = torch.arange(90, total)[:, None]
    j = torch.tensor(places)[None]
    sees = ((j <= i) & (((i - j < window) | (j < sinks)) if window else True)).any(1)
    free = torch.cat([~sees, torch.ones(3, dtype=torch.bool)])
    assert free.sum() > 3
    close(got[free], want[free], tol[free], "rows that do not see it")
    if where == "v" or math.isnan(value):                            # (a score of minus infinity, as an infinite key can give, takes the weight away, and the value with it)
        assert not got[:new][sees].isfinite().all(dim=1).any(), "rows that see it"


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("new,held", [(3, 1), (16, 5), (200, 130), (100, 0)])
def test_rows_in_front_of_position_0_see_nothing(gpu_ctx, new, held, dtype):
    """A batch padded in front: its first rows have no position.  They are zero, and append leaves theirs out."""
    c = Pages([(new, 0), (2, 40)], 2, 2, 128, 16, dtype, 3)
    full_k = c.values("k", 0)
    c.length[0] = held
    out = run(gpu_ctx, c, max_length=500)
    gpu_ctx.check_status()
    assert bool((out[:new - held] == 0).all())
    q = c.q.to(BF).double().view(c.rows, c.kv_heads, c.group, c.dim)[new - held:new]
    if held:
        x = torch.einsum("rhgd,hjd->rhgj", q, full_k[:, :held]) * 128 ** -0.5
        x = x.masked_fill((torch.arange(held)[None] > torch.arange(held)[:, None])[:, None, None], -math.inf)
        want = torch.einsum("rhgj,hjd->rhgd", torch.softmax(x, -1), c.values("v", 0)).reshape(held, -1)
        close(out[new - held:new], want, torch.full_like(want, 0.02), "rows with a position")
    cache, q_out = c.cache(gpu_ctx), torch.full((c.rows, c.heads * c.dim), 77.0, device="cuda")
    before = cache.k.clone()
    cache.append(0, c.batch(gpu_ctx, max_length=500), None, c.x.cuda(), c.heads, q_out)
    gpu_ctx.check_status()
    assert bool((q_out[:new - held] == 77).all()) and torch.equal(q_out[new - held:].cpu(), c.x[new - held:, :c.heads * c.dim])
    touched = (cache.k.view(torch.int8 if dtype == I8 else torch.int16) != before.view(torch.int8 if dtype == I8 else torch.int16)).any(dim=-1).any(dim=2)
    own = torch.zeros_like(touched)
    for s, n in ((0, held), (1, 2)):
        for p in range(int(c.length[s]) - n, int(c.length[s])):
            own[0, int(c.table[s, p // 16]), p % 16] = True
    assert not bool((touched & ~own).any())


@pytest.mark.parametrize("new", [1, 60])
def test_pools_past_32_bit_offsets(gpu_ctx, new):
    """Keys of 4.6 GB: the sequence's pages lie at the end."""
    small = Pages([(new, 300)], 8, 2, 128, 128, I8, 2, layers=1)
    pages = (46 << 27) // (10 * 128 * 8 * 128) * 8
    shape = (1, pages, 8, 128, 128)
    k, v = (torch.zeros(shape, dtype=I8, device="cuda") for _ in "kv")
    ks, vs = (torch.zeros(shape[:4], device="cuda") for _ in "kv")
    assert k.numel() > 1 << 32
    move = pages - small.n_pages
    for t, name in ((k, "k"), (v, "v"), (ks, "k_scale"), (vs, "v_scale")):
        t[:, move:] = getattr(small, name).cuda()
    cache = paged.PagedCache(gpu_ctx, k, v, ks, vs)
    batch = paged.PagedBatch(gpu_ctx, small.start.cuda(), small.length.cuda(), (small.table + move).cuda(), rows=new, max_new=new, max_length=300 + new)
    out = torch.zeros((new, 16 * 128), dtype=F32, device="cuda")
    cache.attend(0, batch, small.q.to(BF).cuda(), 16, out)
    gpu_ctx.check_status()
    want, tol = attention(small, small.q, BF, F32)
    close(out, want, tol)
    # moves: a page and some rows from the end to the front, append at the end
    src = torch.arange(5, dtype=torch.int32, device="cuda") + (pages - 1) * 128
    cache.copy_rows(src, torch.arange(5, dtype=torch.int32, device="cuda"))
    cache.copy_pages(torch.tensor([pages - 1], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda"))
    q = torch.zeros((new, 16 * 128), device="cuda")
    cache.append(0, batch, None, small.x.cuda(), 16, q)
    gpu_ctx.check_status()
    assert torch.equal(k[:, 0, :, :5], small.k[:, -1, :, :5].cuda()) and torch.equal(ks[:, 3].nan_to_num(9), small.k_scale[:, -1].cuda().nan_to_num(9))
    p = 300 + new - 1
    assert torch.equal(vs[0, int(small.table[0, p // 128]) + move, :, p % 128].cpu(), small.x.view(new, -1, 128)[-1, 24:].abs().amax(-1) / 127)


@pytest.mark.parametrize("dtype", [BF, I8])
def test_a_captured_step_follows_the_lengths_on_the_device(gpu_ctx, dtype):
    """Append and attention captured once and replayed while the sequences grow over a page's end; on a stream of its own."""
    c = Pages([(1, 28), (1, 13), (1, 700)], 2, 4, 128, 16, dtype, 5, spare=30)
    spare = [p for p in range(c.n_pages) if p not in c.table.flatten().tolist()]
    table = torch.cat([c.table, torch.tensor(spare[:6], dtype=torch.int32).view(3, 2)], 1)
    for s in range(3):
        table[s, -(-int(c.length[s]) // 16):][:2] = table[s, -2:].clone()
    start, length = c.start.cuda(), c.length.cuda()
    freq = paged.rope_frequencies(128, 10000.0)
    x, q, out = torch.zeros((3, 12 * 128), device="cuda"), torch.zeros((3, 8 * 128), device="cuda"), torch.zeros((3, 8 * 128), device="cuda")

    def make():
        cache = c.cache(gpu_ctx)
        batch = paged.PagedBatch(gpu_ctx, start, length, table.cuda(), rows=3, max_new=1, max_length=800)
        rope = paged.Rope(freq.cuda())

        def step():
            cache.append(0, batch, rope, x, 8, q)
            cache.attend(0, batch, q, 8, out)
        return cache, step

    tokens = [torch.randn((3, 12 * 128), generator=torch.Generator().manual_seed(t)) for t in range(6)]
    results = []
    for captured in (False, True):
        length.copy_(c.length)
        cache, step = make()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            if captured:
                x.copy_(tokens[0].cuda())
                step()
                stream.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    step()
            got = []
            for t in tokens:
                x.copy_(t.cuda())
                g.replay() if captured else step()
                got.append(out.clone())
                length += 1
        stream.synchronize()
        gpu_ctx.check_status()
        results.append((torch.stack(got), cache.k.clone()))
    assert torch.equal(results[0][0], results[1][0])
    assert torch.equal(results[0][1].view(torch.int8), results[1][1].view(torch.int8))
    # the first step against 64 bits: the newest position turned, stored and seen
    c.x = tokens[0]
    heads = turned(tokens[0].view(3, 12, 128)[:, :10], c.length - 1, freq, 128, False).double()
    got = results[0][0][0].view(3, 2, 4, 128).cpu().double()
    for s in range(3):
        k, v = c.values("k", s), c.values("v", s)
        k[:, -1], v[:, -1] = heads[s, 8:10], tokens[0].view(3, 12, 128)[s, 10:].double()
        x64 = torch.einsum("hgd,hjd->hgj", heads[s, :8].view(2, 4, 128), k) * 128 ** -0.5
        want = torch.einsum("hgj,hjd->hgd", torch.softmax(x64, -1), v)
        assert (got[s] - want).abs().max() < 0.03


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("what", ["page", "length", "starts", "rows", "new"])
def test_batches_that_do_not_fit_are_reported(gpu_ctx, what, new, dtype):
    """Nothing outside the arrays is touched (their neighbours keep their values), and the sequences that do fit are right."""
    c = Pages([(new, 100), (new, 40)], 2, 2, 64, 16, dtype, 6)
    bounds = {}
    if what == "page":
        c.table[1, 0] = c.n_pages + 3
        c.table[1, 2] = -5
    elif what == "length":
        c.length[1] = 1 << 20
        bounds = {"max_length": 300}
    elif what == "starts":
        c.start[2] = c.start[1] - 1
    elif what == "rows":
        c.start[2] = 1 << 20
    else:
        c.start[1] = new - 1                                         # the second sequence has a row more than the batch allows
    pad = torch.full((c.rows + 8, c.heads * c.dim), 77.0, device="cuda")
    out = pad[4:-4]
    cache = c.cache(gpu_ctx)
    total = int(c.length[0])
    batch = c.batch(gpu_ctx, max_new=new, max_length=bounds.get("max_length", total), rows=c.rows)
    cache.attend(0, batch, c.q.to(BF).cuda(), c.heads, out)
    with pytest.raises(Hf2qError, match="page"):
        gpu_ctx.check_status()
    assert bool((pad[:4] == 77).all()) and bool((pad[-4:] == 77).all())
    cache.append(0, batch, None, c.x.cuda(), c.heads, out)
    with pytest.raises(Hf2qError, match="page"):
        gpu_ctx.check_status()
    gpu_ctx.check_status()
    assert bool((pad[:4] == 77).all()) and bool((pad[-4:] == 77).all())
    clean = Pages([(new, 100), (new, 40)], 2, 2, 64, 16, dtype, 6)
    cache = clean.cache(gpu_ctx)
    cache.attend(0, batch, c.q.to(BF).cuda(), c.heads, out)
    want, tol = attention(clean, c.q, BF, F32)
    n = new if what != "new" else 0
    close(out[:n], want[:n], tol[:n], "the sequence that fits")
    with pytest.raises(Hf2qError, match="page"):
        gpu_ctx.check_status()
