"""Attention over a paged cache against 64 bits: sizes, layouts and masks where it can go wrong."""
import pytest
import torch

from paged_util import Pages, attention, close

pytestmark = pytest.mark.gpu

BF, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def check(ctx, c, q_dtype=BF, out_dtype=BF, window=0, sinks=0, scale=None, ldq_extra=0, ldo_extra=0, shift=0, **bounds):
    """One call; rows and columns that are not its own stay as they were."""
    q = torch.full((c.rows, c.heads * c.dim + ldq_extra + shift), 9.0).to(q_dtype).cuda()[:, shift:]
    q[:, :c.heads * c.dim] = c.q.to(q_dtype).cuda()
    back = torch.full((c.rows + 3, c.heads * c.dim + ldo_extra + shift), 77.0).to(out_dtype).cuda()
    out = back[:, shift:]
    c.cache(ctx).attend(0, c.batch(ctx, rows=c.rows + 3, **bounds), torch.cat([q, q[:1].expand(3, -1)]) if not (ldq_extra or shift) else _longer(q), c.heads, out, scale=scale,
                        window=window, sinks=sinks)
    ctx.check_status()
    want, tol = attention(c, c.q, q_dtype, out_dtype, scale, window, sinks)
    close(out[:c.rows, :c.heads * c.dim], want, tol)
    assert bool((back[c.rows:] == 77).all()) and bool((back[:, :shift] == 77).all()) and bool((out[:, c.heads * c.dim:] == 77).all())


def _longer(q):
    """The same rows with three more behind them, the distance between rows kept."""
    big = torch.zeros((q.shape[0] + 3, q.stride(0)), dtype=q.dtype, device=q.device)
    view = big[:, q.stride(0) - q.shape[1]:]
    view[:q.shape[0]] = q
    return view


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [[(1, 0)], [(1, 15), (1, 16), (1, 17)], [(1, 127), (1, 128), (1, 700)], [(2, 0)], [(5, 3), (1, 40), (3, 250)], [(33, 0)],
                                     [(129, 1), (1, 300)], [(300, 77)]])
def test_lengths(gpu_ctx, lengths, dim, dtype):
    check(gpu_ctx, Pages(lengths, 2, 4, dim, 16, dtype, 1 + len(lengths)))


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 9, 12, 16, 17, 71])
@pytest.mark.parametrize("new", [1, 4, 40])
def test_groups(gpu_ctx, group, new, dtype):
    check(gpu_ctx, Pages([(new, 90), (1, 7)], 1 if group > 16 else 3, group, 128, 32, dtype, group))


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("new", [1, 70])
def test_pages(gpu_ctx, page, new, dtype):
    check(gpu_ctx, Pages([(new, 1000), (new, page - 1), (new, 0)], 2, 4, 128, page, dtype, page, ld_extra=3))


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (17, 130), (100, 0), (128, 128), (250, 5), (5000, 3)])
@pytest.mark.parametrize("new", [1, 6, 150])
def test_windows(gpu_ctx, new, window, sinks, dtype):
    check(gpu_ctx, Pages([(new, 611), (new, 40), (max(1, new // 2), 0)], 2, 3, 64, 16, dtype, window), window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("q_dtype", [BF, F32])
@pytest.mark.parametrize("out_dtype", [BF, F16, F32])
@pytest.mark.parametrize("new", [1, 65])
def test_types(gpu_ctx, new, out_dtype, q_dtype, dtype):
    check(gpu_ctx, Pages([(new, 333), (1, 5)], 2, 4, 128, 64, dtype, 3), q_dtype, out_dtype)


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("new", [1, 80])
@pytest.mark.parametrize("extra,shift", [(8, 0), (3, 0), (0, 1), (16, 8)])
def test_rows_further_apart_and_off_their_boundaries(gpu_ctx, extra, shift, new, dtype):
    check(gpu_ctx, Pages([(new, 100), (1, 3)], 1, 4, 64, 16, dtype, 4), F32, F16, ldq_extra=extra, ldo_extra=extra, shift=shift)


@pytest.mark.parametrize("dtype", [BF, I8])
def test_sequences_without_new_rows_and_many_of_them(gpu_ctx, dtype):
    lengths = [(0, 50), (1, 9), (0, 0), (3, 64)] + [(s % 3, 5 * s) for s in range(70)] + [(0, 1)]
    check(gpu_ctx, Pages(lengths, 2, 2, 64, 16, dtype, 5))


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("new", [1, 50])
def test_bounds_above_what_the_sequences_hold(gpu_ctx, new, dtype):
    check(gpu_ctx, Pages([(new, 200), (1, 0)], 2, 4, 128, 16, dtype, 6, ld_extra=400), max_new=new, max_length=6000)


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("new,before", [(1, 9000), (3, 20000), (64, 5000), (700, 900)])
def test_long(gpu_ctx, new, before, dtype):
    check(gpu_ctx, Pages([(new, before)], 1, 4, 128, 64, dtype, 7), out_dtype=F16)


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("new", [1, 5, 140])
def test_large_scores(gpu_ctx, new, dtype):
    """The maximum grows along the sequence, by far more than an exponential's range."""
    c = Pages([(new, 500)], 1, 4, 128, 16, dtype, 8)
    ramp = torch.linspace(0.1, 6.0, int(c.length[0]))
    p = torch.arange(int(c.length[0]))
    at = (0, c.table[0, p // 16].long(), slice(None), p % 16)
    if dtype == I8:
        c.k_scale[at] *= ramp[:, None]
        c.v_scale[at] *= (2.0 ** torch.linspace(-20, 20, len(p)))[:, None]         # values of very different sizes
    else:
        c.k[at] = (c.k[at].float() * ramp[:, None, None]).to(BF)
    check(gpu_ctx, c, scale=1.0, out_dtype=F32)
