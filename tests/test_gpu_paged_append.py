"""Rotary turn and append to a paged cache: against 64 bits, and bit for bit against the same steps in 32."""
import pytest
import torch

from hf2q_b200 import paged
from paged_util import STEP, Pages, close, turned

pytestmark = pytest.mark.gpu

BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8


def places(c):
    seq = torch.repeat_interleave(torch.arange(len(c.lengths)), torch.tensor([n for n, _ in c.lengths]))
    pos = torch.cat([torch.arange(b, b + n) for n, b in c.lengths])
    return pos, c.table[seq, pos // c.page].long(), pos % c.page


def run(ctx, c, rot, halves, x_dtype=F32, q_dtype=F32, factor=1.0, layer=0, positions=None, extra=0, theta=10000.0):
    x = torch.zeros((c.rows + 2, c.x.shape[1] + extra), dtype=x_dtype)
    x[:c.rows, :c.x.shape[1]] = c.x.to(x_dtype)
    freq = paged.rope_frequencies(rot, theta) if rot else None
    cache, q = c.cache(ctx), torch.full((c.rows + 2, c.heads * c.dim + extra), 77.0, dtype=q_dtype, device="cuda")
    before = [None if t is None else t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    cache.append(layer, c.batch(ctx, rows=c.rows + 2), paged.Rope(freq.cuda(), halves, factor) if rot else None, x.cuda(), c.heads, q,
                 None if positions is None else positions.cuda())
    ctx.check_status()
    return x[:c.rows, :c.x.shape[1]].float(), freq, cache, q, before


def check(ctx, c, rot, halves, x_dtype=F32, q_dtype=F32, factor=1.0, layer=0, positions=None, extra=0, theta=10000.0):
    x, freq, cache, q, before = run(ctx, c, rot, halves, x_dtype, q_dtype, factor, layer, positions, extra, theta)
    pos, page, row = places(c)
    heads = x.view(c.rows, -1, c.dim)
    h, kv = c.heads, c.kv_heads
    want = heads.double().clone()
    if rot:
        want[:, :h + kv] = turned(heads[:, :h + kv], pos if positions is None else positions[:c.rows], freq, rot, halves, factor)
    # cosine, sine (and their product with factor), two products and a sum: five roundings of terms no larger than |a| + |b|
    size = heads.abs().double() + 1e-30
    if rot:
        size[..., :rot] = heads[..., :rot].abs().double().amax(-1, keepdim=True) * 2 * factor
    tol = 5 * 2.0 ** -24 * size
    close(q[:c.rows, :h * c.dim].view(c.rows, h, c.dim), want[:, :h], tol[:, :h] + (STEP[q_dtype] * 1.01 * want[:, :h].abs() if q_dtype != F32 else 0), "q")
    assert bool((q[c.rows:] == 77).all()) and bool((q[:, h * c.dim:] == 77).all())
    for name, part, old in (("k", slice(h, h + kv), before[0]), ("v", slice(h + kv, h + 2 * kv), before[1])):
        new = getattr(cache, name)
        got = new[layer, page.cuda(), :, row.cuda()].double().cpu()
        if c.dtype == I8:
            scale = getattr(cache, name + "_scale")[layer, page.cuda(), :, row.cuda()].double().cpu()
            unit = want[:, part].abs().amax(-1) / 127
            close(scale, unit, unit * 2.0 ** -22 + 5 * 2.0 ** -24 * size[:, part].amax(-1) / 127, name + "_scale")
            close(got * scale[..., None], want[:, part], 0.501 * unit[..., None] + 8 * 2.0 ** -24 * size[:, part].amax(-1, keepdim=True), name)
        else:
            close(got, want[:, part], tol[:, part] + STEP[BF] * 1.01 * want[:, part].abs() + 2.0 ** -130, name)
        # everything else is as it was
        touched = torch.zeros(new.shape[:4], dtype=torch.bool, device="cuda")
        touched[layer, page.cuda(), :, row.cuda()] = True
        a, b = (t.view(torch.int8 if c.dtype == I8 else torch.int16) for t in (new, old))
        assert bool((a[~touched] == b[~touched]).all())


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("dim,rot,halves", [(128, 128, False), (128, 128, True), (128, 64, True), (128, 10, False), (128, 10, True), (64, 64, True), (64, 64, False), (64, 2, True),
                                            (64, 0, False)])
def test_layouts(gpu_ctx, dim, rot, halves, dtype):
    check(gpu_ctx, Pages([(3, 100), (1, 0), (7, 15)], 2, 3, dim, 16, dtype, rot), rot, halves)


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("x_dtype,q_dtype,extra", [(F32, BF, 0), (BF, F32, 0), (BF, BF, 4), (F32, F32, 3), (BF, BF, 1)])
def test_types_and_strides(gpu_ctx, x_dtype, q_dtype, extra, dtype):
    check(gpu_ctx, Pages([(2, 30), (5, 250)], 3, 1, 128, 32, dtype, 4), 128, True, x_dtype, q_dtype, extra=extra)


@pytest.mark.parametrize("dtype", [BF, I8])
def test_many_sequences_some_idle(gpu_ctx, dtype):
    check(gpu_ctx, Pages([(s % 3, 3 * s) for s in range(100)], 2, 2, 64, 16, dtype, 5), 64, False)


@pytest.mark.parametrize("dtype", [BF, I8])
def test_a_portion_in_the_second_of_three_layers(gpu_ctx, dtype):
    check(gpu_ctx, Pages([(700, 33)], 2, 4, 128, 64, dtype, 6, layers=3), 128, False, factor=1.25, layer=1)


@pytest.mark.parametrize("halves", [False, True])
def test_far_positions(gpu_ctx, halves):
    """At 10^8 an angle in 32 bits would be off by several radians."""
    c = Pages([(6, 2)], 1, 2, 128, 16, BF, 7)
    check(gpu_ctx, c, 128, halves, positions=torch.tensor([0, 1, 12345, 1_000_003, 16_777_217, 100_000_007, 0, 0], dtype=torch.int32), theta=500000.0)


def test_codes_are_the_nearest_whole_numbers(gpu_ctx):
    """Without a turn the codes follow from x alone, bit for bit; a row of zeros has scale 0."""
    c = Pages([(40, 5)], 2, 1, 128, 16, I8, 8)
    c.x[3] = 0
    x, _, cache, _, _ = run(gpu_ctx, c, 0, False)
    _, page, row = places(c)
    for name, heads in (("k", slice(2, 4)), ("v", slice(4, 6))):
        v = x.view(c.rows, -1, 128)[:, heads].numpy()
        top = abs(v).max(-1, keepdims=True)
        unit = (v.dtype.type(127.0) / (top + (top == 0))) * (top > 0)
        assert (getattr(cache, name)[0, page.cuda(), :, row.cuda()].cpu().numpy() == (v * unit).round().astype("int8")).all()
        assert (getattr(cache, name + "_scale")[0, page.cuda(), :, row.cuda()].cpu().numpy() == (top / v.dtype.type(127.0))[..., 0]).all()


def test_scaled_frequencies():
    f = paged.rope_frequencies(128, 500000.0).double()
    assert torch.equal(paged.rope_frequencies(128, 500000.0, linear=4.0).double(), f / 4)
    b = paged.rope_frequencies(128, 500000.0, bands={"factor": 8.0, "low": 1.0, "high": 4.0, "trained": 8192}).double()
    turns = 8192 * f / (2 * torch.pi)
    assert torch.allclose(b[turns < 0.999], f[turns < 0.999] / 8, rtol=1e-6) and torch.equal(b[turns > 4.001], f[turns > 4.001])
    assert bool((b <= f * (1 + 1e-6)).all()) and bool((b >= f / 8 * (1 - 1e-6)).all())
