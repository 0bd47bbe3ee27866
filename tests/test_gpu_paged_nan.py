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
