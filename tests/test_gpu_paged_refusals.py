"""What the paged entries refuse, through the C ABI, before anything is launched; and what is allowed at the edges."""
import ctypes as C

import pytest
import torch

from hf2q_b200 import Hf2qError, _lib, paged
from hf2q_b200.ops import DT_F16
from tests.paged_util import Pages

pytestmark = pytest.mark.gpu


class Call:
    """Arguments of the entries for 3 tokens after 5 in pages of 16, 4 query heads to 2; what a case changes is set on it."""

    def __init__(self, ctx, codes):
        self.ctx = ctx
        self.pages = Pages([(3, 5)], 2, 2, 64, 16, torch.int8 if codes else torch.bfloat16, seed=0)
        self.cache, self.batch = self.pages.cache(ctx), self.pages.batch(ctx)
        self.c = paged._Pages.from_buffer_copy(self.cache.structs[0])
        self.b = paged._PageBatch.from_buffer_copy(self.batch.struct)
        self.freq = paged.rope_frequencies(64, 10000.0).cuda()
        self.r = paged._Rotary(self.freq.data_ptr(), None, 64, 0, 1.0)
        self.x, self.q, self.out = self.pages.x.cuda(), torch.full((3, 256), 7.0, device="cuda"), torch.full((3, 256), 7.0, device="cuda")
        self.scratch = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
        self.a = dict(heads=4, xp=self.x.data_ptr(), xt=0, ldx=512, qp=self.q.data_ptr(), qt=0, ldq=256, op=self.out.data_ptr(), ot=0, ldo=256, sp=self.scratch.data_ptr(),
                      sn=self.scratch.numel(), layers=1, src=torch.zeros(1, dtype=torch.int32, device="cuda"), dst=torch.ones(1, dtype=torch.int32, device="cuda"), n=1)

    def run(self, entry):
        a, h, s, lib = self.a, self.ctx._h, self.ctx._stream(), self.ctx._lib
        c, b, r = (None if t is None else C.byref(t) for t in (self.c, self.b, self.r))
        if entry == "append":
            return lib.hf2q_cuda_pages_append(h, s, c, b, r, a["xp"], a["xt"], a["ldx"], a["heads"], a["qp"], a["qt"], a["ldq"])
        if entry == "attend":
            return lib.hf2q_cuda_pages_attend(h, s, c, b, a["qp"], a["qt"], a["ldq"], a["heads"], 0.125, 0, 0, a["op"], a["ot"], a["ldo"], a["sp"], a["sn"])
        if entry == "bytes":
            return lib.hf2q_cuda_pages_attend_scratch_bytes(h, c, b, a["heads"], 0, 0, C.byref(C.c_uint64()))
        move = lib.hf2q_cuda_pages_copy if entry == "copy" else lib.hf2q_cuda_pages_copy_rows
        at = lambda t: t if t is None else t.data_ptr()
        return move(h, s, c, a["layers"], at(a["src"]), at(a["dst"]), a["n"])


def pages(**kw):
    return lambda t: [setattr(t.c, k, v) for k, v in kw.items()]


def batch(**kw):
    return lambda t: [setattr(t.b, k, v) for k, v in kw.items()]


def rotary(**kw):
    return lambda t: [setattr(t.r, k, v) for k, v in kw.items()]


def args(**kw):
    return lambda t: t.a.update({k: t.a[k] + v[0] if isinstance(v, tuple) else v for k, v in kw.items()})       # (a tuple: added to what is there)


ALL, BATCHES = ("append", "attend", "bytes", "copy", "rows"), ("append", "attend", "bytes")
CASES = [
    (ALL, lambda t: setattr(t, "c", None)), (ALL, pages(k=None)), (ALL, pages(v=None)), (ALL, pages(dtype=0)), (ALL, pages(dtype=9)), (ALL, pages(page=0)), (ALL, pages(page=8)),
    (ALL, pages(page=24)), (ALL, pages(page=512)), (ALL, pages(dim=0)), (ALL, pages(dim=96)), (ALL, pages(dim=256)), (ALL, pages(pages=0)), (ALL, pages(kv_heads=0)),
    (ALL, pages(kv_heads=65536)), (ALL, lambda t: setattr(t.c, "k", t.c.k + 8)), (ALL, lambda t: setattr(t.c, "v", t.c.v + 2)),
    (BATCHES, lambda t: setattr(t, "b", None)), (BATCHES, batch(start=None)), (BATCHES, batch(length=None)), (BATCHES, batch(table=None)), (BATCHES, batch(seqs=0)),
    (BATCHES, batch(seqs=65536)), (BATCHES, batch(table_ld=0)), (BATCHES, batch(max_new=4)), (BATCHES, batch(max_length=2)), (BATCHES, batch(max_length=(1 << 30) + 1)),
    (BATCHES, batch(rows=(1 << 28) + 1)),
    (("attend", "bytes"), args(heads=0)), (("attend", "bytes"), args(heads=3)), (("attend", "bytes"), args(heads=65536)), (("attend", "bytes"), args(heads=2 * 129)),
    (("append",), args(heads=65536)), (("append",), args(xp=None)), (("append", "attend"), args(qp=None)), (("attend",), args(op=None)), (("append",), args(xt=DT_F16)), (("append",), args(xt=7)),
    (("append", "attend"), args(qt=DT_F16)), (("append", "attend"), args(qt=3)), (("attend",), args(ot=3)), (("append",), args(ldx=511)), (("append", "attend"), args(ldq=255)),
    (("attend",), args(ldo=255)), (("append",), args(xp=(2,))), (("append", "attend"), args(qp=(1,))), (("attend",), args(op=(2,))), (("attend",), args(sp=(128,))),
    (("append",), rotary(rot_dim=63)), (("append",), rotary(rot_dim=66)), (("append",), rotary(freq=None)),
    (("copy", "rows"), args(layers=0)), (("copy", "rows"), args(layers=65536)), (("copy", "rows"), args(src=None)), (("copy", "rows"), args(dst=None)), (("copy",), args(n=0x80000000)),
]


@pytest.mark.parametrize("codes", [True, False], ids=["codes", "bf16"])
def test_entries_refuse_what_they_are_not_for(gpu_ctx, codes):
    for i, (entries, change) in enumerate(CASES):
        for entry in entries:
            t = Call(gpu_ctx, codes)
            change(t)
            rc = t.run(entry)
            assert rc == _lib.ERR_INVALID_ARGUMENT, (i, entry, rc)
            with pytest.raises(Hf2qError):
                gpu_ctx._check(rc)
            assert bool((t.out == 7).all()) and bool((t.q == 7).all())
    gpu_ctx.check_status()


def test_codes_need_scales_and_parts_need_scratch(gpu_ctx):
    for name in ("k_scale", "v_scale"):
        for entry in ALL:
            t = Call(gpu_ctx, True)
            setattr(t.c, name, None)
            assert t.run(entry) == _lib.ERR_INVALID_ARGUMENT
            t = Call(gpu_ctx, True)
            setattr(t.c, name, getattr(t.c, name) + 4)
            assert t.run(entry) == _lib.ERR_INVALID_ARGUMENT
    t = Call(gpu_ctx, True)
    need = C.c_uint64()
    gpu_ctx._check(gpu_ctx._lib.hf2q_cuda_pages_attend_scratch_bytes(gpu_ctx._h, C.byref(t.c), C.byref(t.b), 4, 0, 0, C.byref(need)))
    assert need.value > 0
    assert gpu_ctx._lib.hf2q_cuda_pages_attend_scratch_bytes(gpu_ctx._h, C.byref(t.c), C.byref(t.b), 4, 0, 0, None) == _lib.ERR_INVALID_ARGUMENT
    for change in (dict(sp=None), dict(sn=need.value - 1), dict(sn=0)):
        t = Call(gpu_ctx, True)
        t.a.update(change)
        assert t.run("attend") == _lib.ERR_WORKSPACE
    gpu_ctx.check_status()


def test_calls_without_rows_or_places_do_nothing(gpu_ctx):
    for entry, change in (("append", batch(rows=0, max_new=0)), ("attend", batch(rows=0, max_new=0)), ("attend", batch(max_new=0)), ("copy", args(n=0, src=None, dst=None)),
                          ("rows", args(n=0, src=None, dst=None))):
        t = Call(gpu_ctx, True)
        k = t.cache.k.clone()
        change(t)
        assert t.run(entry) == 0
        assert bool((t.out == 7).all()) and bool((t.q == 7).all()) and torch.equal(k, t.cache.k)
    gpu_ctx.check_status()


def test_the_classes_refuse_too(gpu_ctx):
    t = Call(gpu_ctx, True)
    cache, batch_, rope = t.cache, t.batch, paged.Rope(t.freq)
    bad = [
        lambda: cache.append(1, batch_, rope, t.x, 4, t.q), lambda: cache.append(-1, batch_, rope, t.x, 4, t.q), lambda: cache.append(0, batch_, rope, t.x[:2], 4, t.q),
        lambda: cache.append(0, batch_, rope, t.x.half(), 4, t.q), lambda: cache.append(0, batch_, rope, t.x.t(), 4, t.q), lambda: cache.append(0, batch_, rope, t.x.cpu(), 4, t.q),
        lambda: cache.append(0, batch_, rope, t.x, 4, t.q.half()), lambda: cache.append(0, batch_, rope, t.x, 4, t.q, positions=torch.zeros(2, dtype=torch.int32, device="cuda")),
        lambda: cache.append(0, batch_, rope, t.x, 4, t.q, positions=torch.zeros(3, device="cuda")), lambda: cache.attend(0, batch_, t.q, 3, t.out),
        lambda: cache.attend(0, batch_, t.q, 4, t.out, window=-1), lambda: cache.attend(0, batch_, t.q, 4, t.out, sinks=-1), lambda: cache.attend(0, batch_, t.q[:, :255], 4, t.out),
        lambda: cache.attend(0, batch_, t.q[:1].expand(3, 256), 4, t.out), lambda: cache.attend(0, batch_, t.q, 4, t.out.double()),
        lambda: cache.copy_pages(torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")),
        lambda: cache.copy_rows(torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda")),
        lambda: paged.PagedCache(gpu_ctx, cache.k, cache.v), lambda: paged.PagedCache(gpu_ctx, cache.k, cache.v[:, :1], cache.k_scale, cache.v_scale),
        lambda: paged.PagedCache(gpu_ctx, cache.k, cache.v, cache.k_scale, cache.v_scale[..., :8]), lambda: paged.PagedCache(gpu_ctx, cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0]),
        lambda: t.pages.batch(gpu_ctx, max_new=9, rows=3), lambda: t.pages.batch(gpu_ctx, max_length=2), lambda: t.pages.batch(gpu_ctx, max_length=1 << 32),
        lambda: t.pages.batch(gpu_ctx, rows=(1 << 32) + 3), lambda: cache.attend(0, batch_, t.q, 4, t.out, window=1 << 32), lambda: cache.attend(0, batch_, t.q, 4, t.out, sinks=1 << 32),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(Hf2qError):
            call()
            pytest.fail(f"case {i} was taken")
    assert bool((t.out == 7).all()) and bool((t.q == 7).all())
    gpu_ctx.check_status()
