"""Calls over pages at the edges of what is allowed: no rows."""
import pytest
import torch

from hf2q_b200 import paged
from tests.paged_util import Pages

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
