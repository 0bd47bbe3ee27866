"""Infinite and NaN values in blocks of positions that follow one another, each seen by some of the rows: what blocks before gave has to be
there when a row adds such values up by itself, or it is lost, also for elements that are finite."""
import math

import pytest
import torch

from tests.paged_util import Pages, attention, close

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
AT = {0: 3, 1: 17}                                                    # the element of each KV head that is bad


# (new, before, group, dim, window, sinks): one and several partly seen blocks, one and two tiles, positions in parts, a window's both ends, few rows
@pytest.mark.parametrize("new,before,group,dim,window,sinks", [(256, 10, 1, 128, 0, 0), (200, 700, 2, 64, 0, 0), (150, 90, 2, 128, 0, 0), (300, 5, 1, 64, 100, 3),
                                                               (180, 300, 2, 128, 130, 70), (64, 5000, 4, 128, 0, 0), (128, 3000, 2, 64, 1500, 0), (7, 40, 2, 128, 0, 0)])
@pytest.mark.parametrize("values", [(math.nan,), (math.inf, -math.inf, math.nan)], ids=["nan", "mixed"])
def test_finite_elements_are_right_beside_bad_ones(gpu_ctx, values, new, before, group, dim, window, sinks):
    c, clean = (Pages([(new, before), (2, 9)], 2, group, dim, 16, BF, new + before) for _ in "ab")
    total = before + new
    first = max(0, before - window) + 5 if window else before + 5
    bad = torch.arange(first, first + 60 if window else total, 13)                                      # (a window: the last rows have left them behind)
    for n, p in enumerate(bad.tolist()):
        for head, d in AT.items():
            c.v[0, int(c.table[0, p // 16]), head, p % 16, d] = values[n % len(values)]
    cache, batch, q = c.cache(gpu_ctx), c.batch(gpu_ctx), c.q.to(BF).cuda()
    want, tol = attention(clean, c.q, BF, F32, None, window, sinks)
    i, j = torch.arange(before, total)[:, None], bad[None]
    sees = ((j <= i) & (((i - j < window) | (j < sinks)) if window else True)).any(1)
    assert 3 < int((~sees).sum()) or new < 16
    mask = torch.zeros((c.rows, 2, group, dim), dtype=torch.bool)     # what a bad value reaches
    for head, d in AT.items():
        mask[:new, head, :, d] = sees[:, None]
    mask = mask.view(c.rows, -1)
    for _ in range(5):
        out = torch.full((c.rows, c.heads * dim), 77.0, device="cuda")
        cache.attend(0, batch, q, c.heads, out, window=window, sinks=sinks)
        gpu_ctx.check_status()
        got = out.cpu().double()
        assert not bool(got[mask].isfinite().any())
        close(got[~mask], want[~mask], tol[~mask], "elements that no bad value reaches")
