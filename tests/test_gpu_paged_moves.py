"""Pages and single rows of a paged cache, moved: every byte, in all layers, and nothing else."""
import pytest
import torch

from hf2q_b200 import Hf2qError
from paged_util import Pages

pytestmark = pytest.mark.gpu

BF, I8 = torch.bfloat16, torch.int8


def arrays(cache):
    return [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]


def bits(t):
    return t.view({1: torch.int8, 2: torch.int16, 4: torch.int32}[t.element_size()])


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("dim,page,kv_heads", [(128, 16, 8), (64, 16, 1), (64, 128, 3), (128, 256, 5)])
@pytest.mark.parametrize("layers,n", [(1, 1), (3, 7)])
def test_whole_pages(gpu_ctx, layers, n, dim, page, kv_heads, dtype):
    c = Pages([(1, 20 * page - 1)], kv_heads, 1, dim, page, dtype, n, layers=layers)
    cache, order = c.cache(gpu_ctx), torch.randperm(c.n_pages, generator=torch.Generator().manual_seed(n))
    src, dst = order[:n], order[n:2 * n]
    want = [t.clone().index_copy_(1, dst.cuda(), t[:, src.cuda()]) for t in arrays(cache)]
    cache.copy_pages(src.int().cuda(), dst.int().cuda())
    gpu_ctx.check_status()
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(arrays(cache), want))


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("dim,page,kv_heads", [(128, 16, 8), (64, 32, 1), (64, 128, 3), (128, 256, 2)])
@pytest.mark.parametrize("layers,n", [(1, 1), (2, 37), (1, 900)])
def test_single_rows(gpu_ctx, layers, n, dim, page, kv_heads, dtype):
    c = Pages([(1, 2047)], kv_heads, 1, dim, page, dtype, n, layers=layers)
    cache, order = c.cache(gpu_ctx), torch.randperm(c.n_pages * page, generator=torch.Generator().manual_seed(n))
    src, dst = order[:n], order[n:2 * n]
    want = []
    for t in arrays(cache):
        w = t.clone()
        w[:, (dst // page).cuda(), :, (dst % page).cuda()] = t[:, (src // page).cuda(), :, (src % page).cuda()]
        want.append(w)
    cache.copy_rows(src.int().cuda(), dst.int().cuda())
    gpu_ctx.check_status()
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(arrays(cache), want))


@pytest.mark.parametrize("dtype", [BF, I8])
@pytest.mark.parametrize("move", ["copy_pages", "copy_rows"])
def test_numbers_out_of_range_move_nothing(gpu_ctx, move, dtype):
    c = Pages([(1, 63)], 2, 1, 64, 16, dtype, 3)
    cache, most = c.cache(gpu_ctx), c.n_pages * (16 if move == "copy_rows" else 1)
    before = [t.clone() for t in arrays(cache)]
    getattr(cache, move)(torch.tensor([most, 0, -1], dtype=torch.int32).cuda(), torch.tensor([1, most + 5, 2], dtype=torch.int32).cuda())
    with pytest.raises(Hf2qError, match="page"):
        gpu_ctx.check_status()
    gpu_ctx.check_status()
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(arrays(cache), before))


def test_nothing_to_move(gpu_ctx):
    cache = Pages([(1, 63)], 2, 1, 64, 16, I8, 3).cache(gpu_ctx)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    cache.copy_pages(none, none)
    cache.copy_rows(none, none)
    gpu_ctx.check_status()
