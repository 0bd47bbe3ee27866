"""A NaN that goes into paged attention comes out of it, in every type of result, and a NaN that is appended stays one."""
import math

import pytest
import torch

from tests.paged_util import Pages, attention, close

pytestmark = pytest.mark.gpu

BF, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def attend(ctx, c, q, out_dtype):
    out = torch.full((c.rows, c.heads * c.dim), 7.0, dtype=out_dtype, device="cuda")
    c.cache(ctx).attend(0, c.batch(ctx), q.cuda(), c.heads, out)
    ctx.check_status()
    return out.cpu().view(c.rows, c.kv_heads, c.group, c.dim)


# one and several parts of few and of many rows
@pytest.mark.parametrize("new,before", [(1, 60), (1, 5000), (7, 300), (200, 100), (64, 5000)])
@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("out_dtype", [F32, BF, F16])
@pytest.mark.parametrize("where", ["q", "k", "v"])
def test_nan_comes_out(gpu_ctx, where, out_dtype, dtype, new, before):
    c, clean = (Pages([(new, before), (2, 30)], 2, 4, 128, 16, dtype, 11) for _ in "ab")
    q, reached = c.q.clone(), torch.zeros((c.rows, 2, 4, 128), dtype=torch.bool)
    if where == "q":
        q[new - 1, 128 * 5 + 9] = math.nan                            # head 1 of KV head 1
        reached[new - 1, 1, 1] = True
    elif dtype == I8:
        getattr(c, where + "_scale")[0, int(c.table[0, 0]), 1, 3] = math.nan
        reached[:new, 1] = True
    else:
        getattr(c, where)[0, int(c.table[0, 0]), 1, 3, 9] = math.nan
        reached[:new, 1, :, slice(9, 10) if where == "v" else slice(None)] = True
    got = attend(gpu_ctx, c, q, out_dtype)
    assert bool(got[reached].isnan().all())
    want, tol = attention(clean, clean.q, F32, out_dtype)
    close(got[~reached], want.view(got.shape)[~reached], tol.view(got.shape)[~reached], "what it does not reach")


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("rot", [0, 64])
def test_nan_that_is_appended_stays(gpu_ctx, rot, dtype):
    """A key and a value with a NaN: attention over them gives NaN, the other heads and positions are numbers."""
    from hf2q_b200 import paged
    c = Pages([(4, 20), (1, 3)], 2, 2, 128, 16, dtype, 12)
    heads = c.x.view(c.rows, -1, 128)
    heads[1, 4, 100] = math.nan                                       # key head 0 of the second row (in front of it the queries), not among what is turned
    heads[2, 7, 5] = -math.nan                                        # value head 1 of the third
    cache, q = c.cache(gpu_ctx), torch.empty((c.rows, c.heads * 128), device="cuda")
    cache.append(0, c.batch(gpu_ctx), paged.Rope(paged.rope_frequencies(rot, 10000.0).cuda()) if rot else None, c.x.cuda(), c.heads, q)
    gpu_ctx.check_status()
    value = lambda t, scale: t.double() * (1 if scale is None else scale.double()[..., None])
    for t, name, row, head, d in ((value(cache.k, cache.k_scale), "k", 1, 0, 100), (value(cache.v, cache.v_scale), "v", 2, 1, 5)):
        for r in range(4):
            p = 20 + r
            got = t[0, int(c.table[0, p // 16]), :, p % 16].cpu()
            bad = torch.zeros((2, 128), dtype=torch.bool)
            if r == row:
                bad[head, slice(None) if dtype == I8 else d] = True
            assert torch.equal(got.isnan(), bad), (name, r)
    out = torch.empty((c.rows, c.heads * 128), device="cuda")
    cache.attend(0, c.batch(gpu_ctx), q, c.heads, out)
    gpu_ctx.check_status()
    nan = out.cpu().view(c.rows, 2, 2, 128).isnan()
    want = torch.zeros_like(nan)
    want[1:4, 0] = True                                               # rows from the second on see the key
    want[2:4, 1, :, slice(None) if dtype == I8 else 5] = True         # from the third on the value
    assert torch.equal(nan, want)
