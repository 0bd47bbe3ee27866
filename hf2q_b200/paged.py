"""A key-value cache in pages, for many sequences: ctypes view of the ``pages`` entries of the C ABI and the host side of the pool.

``PagedCache`` holds the pages of one or several layers and launches the entries on torch's current stream; ``PagedBatch`` names the
sequences of a call by arrays on the device; ``Rope`` is a model's rotary turn; ``PagePool`` keeps, on the host, which sequence owns
which page: it hands pages out, shares them between branches of a sequence, and packs and frees them.
"""
from __future__ import annotations

import ctypes as C
import heapq
import math
from contextlib import nullcontext
from functools import wraps

import torch

from . import _lib, ops
from .ops import _TORCH_DT, DT_BF16, Hf2qError

DT_I8 = 3
_vp, _u32, _f32 = C.c_void_p, C.c_uint32, C.c_float


class _Pages(C.Structure):             # hf2q_pages in include/hf2q_cuda.h
    _fields_ = [(n, _vp) for n in ("k", "v", "k_scale", "v_scale")] + [(n, _u32) for n in ("pages", "page", "kv_heads", "dim", "dtype")]


class _PageBatch(C.Structure):         # hf2q_page_batch
    _fields_ = [(n, _vp) for n in ("start", "length", "table")] + [(n, _u32) for n in ("seqs", "rows", "table_ld", "max_new", "max_length")]


class _Rotary(C.Structure):            # hf2q_rotary
    _fields_ = [("freq", _vp), ("pos", _vp), ("rot_dim", _u32), ("halves", _u32), ("factor", _f32)]


def _refuse(text: str):
    raise Hf2qError(_lib.ERR_INVALID_ARGUMENT, text)


def _on_device(t: torch.Tensor, name: str, dtypes, ctx, contiguous: bool = True) -> None:
    if t.dtype not in dtypes:
        _refuse(f"{name} dtype {t.dtype} (want {' or '.join(str(d) for d in dtypes)})")
    if not t.is_cuda or t.device.index != ctx.device or (contiguous and not t.is_contiguous()):
        _refuse(f"{name} must be a {'contiguous ' if contiguous else ''}tensor on cuda:{ctx.device}")


def _rows(t: torch.Tensor, name: str, dtypes, rows: int, width: int, ctx) -> int:
    """Checks a matrix whose rows may lie further apart than they are wide; returns their distance.  (On the way of every call: what is
    right is seen with few questions.)"""
    if t.dtype in dtypes and t.get_device() == ctx.device and t.dim() == 2:
        (n, w), (ld, one) = t.shape, t.stride()
        if n >= rows and w >= width and (one == 1 or w <= 1) and (rows <= 1 or width <= ld < 1 << 32):
            return ld if rows > 1 else width
    _on_device(t, name, dtypes, ctx, contiguous=False)
    _refuse(f"{name} must hold {rows} rows of {width} elements side by side")


_INT = (torch.int32, torch.uint32)
_IN, _OUT = (torch.float32, torch.bfloat16), (torch.float32, torch.bfloat16, torch.float16)


def rope_frequencies(rot_dim: int, theta: float, *, linear: float = 1.0, bands: dict | None = None) -> torch.Tensor:
    """theta^(-2i / rot_dim) radians a position, f32 [rot_dim / 2], scaled for contexts longer than a model was trained on: all of them divided
    by ``linear``, or with ``bands`` = {"factor", "low", "high", "trained"} only those whose wavelength is long against the trained
    context: above trained / low they are divided by factor, below trained / high kept, in between in proportion."""
    f = theta ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim) / linear
    if bands:
        turns = bands["trained"] * f / (2 * math.pi)                   # of the trained context
        keep = ((turns - bands["low"]) / (bands["high"] - bands["low"])).clamp(0, 1)
        f = f * (keep + (1 - keep) / bands["factor"])
    return f.to(torch.float32)


class Rope:
    """A model's rotary turn: ``freq`` f32 [pairs] on the device; pairs side by side, or the two halves of the turned part; ``factor``
    multiplies what is turned."""

    def __init__(self, freq: torch.Tensor, halves: bool = False, factor: float = 1.0):
        if freq.dtype != torch.float32 or not freq.is_cuda or not freq.is_contiguous() or freq.dim() != 1:
            _refuse("freq must be a contiguous float32 vector on the device")
        self.freq, self.halves, self.factor, self.device = freq, bool(halves), float(factor), freq.get_device()
        self._plain = self.struct(None)
        self.ref = C.byref(self._plain)

    def struct(self, positions: torch.Tensor | None) -> _Rotary:
        return _Rotary(self.freq.data_ptr(), None if positions is None else positions.data_ptr(), 2 * self.freq.numel(), int(self.halves), self.factor)


class PagedBatch:
    """The sequences of a call (see hf2q_page_batch): ``start`` [seqs + 1], ``length`` [seqs] and ``table`` [seqs, pages] on the device, and
    host-side bounds that the launches are laid out for.  The arrays may change between calls within the bounds.  The scratch of
    attention calls belongs to the batch: calls on the same batch follow one another on one stream."""

    def __init__(self, ctx: ops.GpuContext, start: torch.Tensor, length: torch.Tensor, table: torch.Tensor, *, rows: int, max_new: int, max_length: int):
        _on_device(start, "start", _INT, ctx)
        _on_device(length, "length", _INT, ctx)
        _on_device(table, "table", _INT, ctx, contiguous=False)
        seqs = length.numel()
        if length.dim() != 1 or start.dim() != 1 or table.dim() != 2 or start.numel() != seqs + 1 or table.shape[0] != seqs or seqs == 0 or table.shape[1] == 0:
            _refuse("a batch of n sequences has n + 1 starts, n lengths and n rows of page numbers")
        if table.stride(1) != 1 and table.shape[1] > 1 or seqs > 1 and table.stride(0) < table.shape[1]:
            _refuse("the page numbers of a sequence lie side by side")
        if not 0 <= max_new <= rows <= 1 << 28 or not max_new <= max_length <= 1 << 30:
            _refuse("max_new is at most rows (2^28) and at most max_length (2^30)")
        self.ctx, self._keep = ctx, (start, length, table)
        self.rows, self.max_new, self.max_length = int(rows), int(max_new), int(max_length)
        self.struct = _PageBatch(start.data_ptr(), length.data_ptr(), table.data_ptr(), seqs, self.rows, table.stride(0) if seqs > 1 else table.shape[1],
                                 self.max_new, self.max_length)
        self.ref, self._scratch = C.byref(self.struct), {}

    def scratch(self, pages: _Pages, heads: int, window: int, sinks: int) -> torch.Tensor:
        """Scratch of attention calls of these sizes."""
        key = (pages.kv_heads, pages.dim, pages.dtype, pages.page, heads, window, sinks)
        buf = self._scratch.get(key)
        if buf is None:
            need = C.c_uint64()
            self.ctx._check(self.ctx._lib.hf2q_cuda_pages_attend_scratch_bytes(self.ctx._h, C.byref(pages), self.ref, heads, window, sinks, C.byref(need)))
            buf = self._scratch[key] = torch.empty(max(need.value, 256), dtype=torch.uint8, device=torch.device("cuda", self.ctx.device))
        return buf


class PagedCache:
    """Pages of ``layers`` layers: k, v [layers, pages, kv_heads, page, dim], bf16, or int8 with f32 scales [layers, pages, kv_heads, page]."""

    def __init__(self, ctx: ops.GpuContext, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
        for t, name in ((k, "k"), (v, "v")):
            _on_device(t, name, (torch.bfloat16, torch.int8), ctx)
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype or k.shape[0] == 0:
            _refuse("k and v are [layers, pages, kv_heads, page, dim] of one type")
        codes = k.dtype == torch.int8
        if codes != (k_scale is not None) or codes != (v_scale is not None):
            _refuse("int8 pages have scales, bfloat16 pages have none")
        if codes:
            for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
                _on_device(t, name, (torch.float32,), ctx)
                if t.shape != k.shape[:4]:
                    _refuse(f"{name} must be [layers, pages, kv_heads, page]")
        self.ctx, self.k, self.v, self.k_scale, self.v_scale = ctx, k, v, k_scale, v_scale
        self.layers, self.pages, self.kv_heads, self.page, self.dim = k.shape
        step = lambda t: 0 if t is None else t.stride(0) * t.element_size()
        first = [(0 if t is None else t.data_ptr(), step(t)) for t in (k, v, k_scale, v_scale)]
        self.structs = [_Pages(*(p + i * n or None for p, n in first), self.pages, self.page, self.kv_heads, self.dim, DT_I8 if codes else DT_BF16) for i in range(self.layers)]
        self._refs, self._scale = [C.byref(s) for s in self.structs], self.dim ** -0.5
        self._append, self._attend = ctx._lib.hf2q_cuda_pages_append, ctx._lib.hf2q_cuda_pages_attend

    @classmethod
    def allocate(cls, ctx: ops.GpuContext, layers: int, pages: int, page: int, kv_heads: int, dim: int, dtype=torch.int8) -> "PagedCache":
        dev = torch.device("cuda", ctx.device)
        kv = [torch.zeros((layers, pages, kv_heads, page, dim), dtype=dtype, device=dev) for _ in "kv"]
        scales = [torch.zeros((layers, pages, kv_heads, page), dtype=torch.float32, device=dev) for _ in "kv"] if dtype == torch.int8 else [None, None]
        return cls(ctx, *kv, *scales)

    def _check(self, layer: int, batch: PagedBatch) -> None:
        if not 0 <= layer < self.layers:
            _refuse(f"layer {layer} of {self.layers}")
        if batch.ctx is not self.ctx:
            _refuse("the batch belongs to another context")

    def append(self, layer: int, batch: PagedBatch, rope: Rope | None, x: torch.Tensor, heads: int, q_out: torch.Tensor, positions: torch.Tensor | None = None) -> None:
        """Rows of x [rows, (heads + 2 kv_heads) * dim] (queries, keys, values): turned queries to q_out [rows, heads * dim], turned keys and the
        values to the layer's pages.  ``positions`` [rows]: turn by these instead of the positions in the sequences."""
        ctx, rows = self.ctx, batch.rows
        self._check(layer, batch)
        ldx = _rows(x, "x", _IN, rows, (heads + 2 * self.kv_heads) * self.dim, ctx)
        ldq = _rows(q_out, "q_out", _IN, rows, heads * self.dim, ctx)
        if positions is not None:
            _on_device(positions, "positions", _INT, ctx)
            if positions.numel() < batch.rows:
                _refuse(f"positions must hold {batch.rows} numbers")
        if rope is not None and rope.device != ctx.device:
            _refuse(f"freq must be on cuda:{ctx.device}")
        turn = None if rope is None else rope.ref if positions is None else C.byref(rope.struct(positions))
        rc = self._append(ctx._h, ctx._stream(), self._refs[layer], batch.ref, turn, x.data_ptr(), _TORCH_DT[x.dtype], ldx, heads, q_out.data_ptr(), _TORCH_DT[q_out.dtype], ldq)
        if rc:
            ctx._check(rc)

    def attend(self, layer: int, batch: PagedBatch, q: torch.Tensor, heads: int, out: torch.Tensor, scale: float | None = None, window: int = 0, sinks: int = 0) -> None:
        """out [rows, heads * dim] = attention of q's rows over their sequences (``scale`` None: dim^-1/2; ``window`` 0: all positions before)."""
        ctx, rows, width = self.ctx, batch.rows, heads * self.dim
        self._check(layer, batch)
        ldq, ldo = _rows(q, "q", _IN, rows, width, ctx), _rows(out, "out", _OUT, rows, width, ctx)
        if not (0 <= window < 1 << 32 and 0 <= sinks < 1 << 32):
            _refuse("window and sinks are not negative, and below 2^32")
        scratch = batch.scratch(self.structs[layer], heads, window, sinks)
        rc = self._attend(ctx._h, ctx._stream(), self._refs[layer], batch.ref, q.data_ptr(), _TORCH_DT[q.dtype], ldq, heads, self._scale if scale is None else scale, window, sinks,
                          out.data_ptr(), _TORCH_DT[out.dtype], ldo, scratch.data_ptr(), scratch.numel())
        if rc:
            ctx._check(rc)

    def _move(self, entry: str, src: torch.Tensor, dst: torch.Tensor) -> None:
        ctx = self.ctx
        _on_device(src, "src", _INT, ctx)
        _on_device(dst, "dst", _INT, ctx)
        if src.numel() != dst.numel():
            _refuse("src and dst name as many places")
        ctx._check(getattr(ctx._lib, entry)(ctx._h, ctx._stream(), self._refs[0], self.layers, src.data_ptr(), dst.data_ptr(), src.numel()))

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Pages src[i] -> dst[i] of all layers; no destination is a source or named twice."""
        self._move("hf2q_cuda_pages_copy", src, dst)

    def copy_rows(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Rows src[i] -> dst[i] of all layers (row r of page g is g * page + r); no destination is a source or named twice."""
        self._move("hf2q_cuda_pages_copy_rows", src, dst)


def _shifted(runs: list, keep: list) -> list:
    """The runs (first place, position - place) of a sequence of which the places ``keep`` are left."""
    out, k = [], 0
    for i, p in enumerate(keep):
        while k + 1 < len(runs) and runs[k + 1][0] <= p:
            k += 1
        shift = runs[k][1] + p - i
        if not out or out[-1][1] != shift:
            out.append((i, shift))
    return out or [(0, 0)]


def _in_order(method):
    @wraps(method)
    def call(self, *args, **kw):
        with self._ordered():
            return method(self, *args, **kw)
    return call


class PagePool:
    """Which sequence owns which pages of a cache, kept on the host: pages are handed out lowest number first, branches of a sequence share
    them, and a shared page is copied before one of its owners writes into it.

    ``table`` [seqs, pages of max_length] and ``length`` [seqs] on the device follow the books, in the order of the current stream, for
    ``PagedBatch`` to read.

    ``compact`` leaves keys turned by the positions that they had.  A sequence's next token is then turned by the position behind its last
    key's, ``length_of + shift_of``, and not by its place (``append``'s ``positions``); ``shift`` [seqs] says so on the device.

    ``ordered``: a context manager that every call which reaches the device runs in, for owners whose calls come on several streams."""

    def __init__(self, cache: PagedCache, seqs: int, max_length: int, ordered=nullcontext):
        if seqs < 1 or max_length < 1:
            _refuse("a pool serves 1 sequence or more, of 1 position or more")
        self.cache, self.seqs, self.max_length, self._ordered = cache, seqs, max_length, ordered
        dev = cache.k.device
        self.table = torch.full((seqs, -(-max_length // cache.page)), -1, dtype=torch.int32, device=dev)
        self.length = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self.shift = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self._free, self._refs = list(range(cache.pages)), [0] * cache.pages             # (a heap)
        self._pages: list = [None] * seqs                                                # page numbers of an open sequence
        self._lengths = [0] * seqs
        self._shifts: list = [[(0, 0)] for _ in range(seqs)]                             # runs (first place, position - place), up to the next run's first place

    # ---- what the books say
    @property
    def n_free_pages(self) -> int:
        return len(self._free)

    def pages_of(self, seq: int) -> list:
        return list(self._own(seq))

    def length_of(self, seq: int) -> int:
        self._own(seq)
        return self._lengths[seq]

    def shift_of(self, seq: int) -> int:
        """How far the position that the sequence's next token is turned by lies behind its place."""
        self._own(seq)
        return self._shifts[seq][-1][1]

    def _own(self, seq: int) -> list:
        if not 0 <= seq < self.seqs or self._pages[seq] is None:
            raise RuntimeError(f"sequence {seq} is not in use")
        return self._pages[seq]

    def _vacant(self) -> int:
        for s, p in enumerate(self._pages):
            if p is None:
                return s
        raise RuntimeError("no free sequence slot")

    def _take(self, n: int) -> list:
        if n > len(self._free):
            raise RuntimeError(f"no free page ({n} wanted, {len(self._free)} of {self.cache.pages} free)")
        out = [heapq.heappop(self._free) for _ in range(n)]
        for p in out:
            self._refs[p] = 1
        return out

    def _drop(self, pages) -> None:
        for p in pages:
            self._refs[p] -= 1
            if self._refs[p] == 0:
                heapq.heappush(self._free, p)

    def _numbers(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).to(self.table.device)

    def _publish(self, seq: int) -> None:
        """The device's row and length; a place without a page holds -1, which the entries report and skip."""
        pages = self._pages[seq] or []
        if pages:
            self.table[seq, :len(pages)] = self._numbers(pages)
        self.table[seq, len(pages):].fill_(-1)
        self.length[seq:seq + 1].fill_(self._lengths[seq])
        self.shift[seq:seq + 1].fill_(self._shifts[seq][-1][1])

    # ---- sequences
    @_in_order
    def open(self) -> int:
        """A new sequence without positions."""
        seq = self._vacant()
        self._pages[seq], self._lengths[seq], self._shifts[seq] = [], 0, [(0, 0)]
        self._publish(seq)
        return seq

    @_in_order
    def close(self, seq: int) -> None:
        """Gives the sequence's pages back, as far as no branch shares them."""
        self._drop(self._own(seq))
        self._pages[seq], self._lengths[seq], self._shifts[seq] = None, 0, [(0, 0)]
        self._publish(seq)

    @_in_order
    def reserve(self, seq: int, n: int) -> None:
        """Pages of its own for the sequence's next n positions (which ``advance`` then counts)."""
        pages, size, have = self._own(seq), self.cache.page, self._lengths[seq]
        if n < 0 or have + n > self.max_length:
            _refuse(f"{n} positions after {have}: the pool holds sequences of up to {self.max_length}")
        if n == 0:
            return
        first = have // size
        shared = [i for i in range(first, len(pages)) if self._refs[pages[i]] > 1]       # pages that will be written into
        new = self._take(len(shared) + max(0, -(-(have + n) // size) - len(pages)))
        if shared:
            used = [i for i in shared if i * size < have]                                # only the one that is partly filled holds anything
            if used:
                self.cache.copy_pages(self._numbers([pages[i] for i in used]), self._numbers(new[:len(used)]))
            old = [pages[i] for i in shared]
            for i, p in zip(shared, new):
                pages[i] = p
            self._drop(old)
        pages += new[len(shared):]
        if new:
            self.table[seq, first:len(pages)] = self._numbers(pages[first:])

    @_in_order
    def advance(self, seq: int, n: int) -> None:
        """The sequence has n more positions, in pages that ``reserve`` gave it."""
        pages, total = self._own(seq), self._lengths[seq] + n
        if n < 0 or total > min(len(pages) * self.cache.page, self.max_length):
            _refuse(f"{n} positions were not reserved")
        self._lengths[seq] = total
        self.length[seq:seq + 1].fill_(total)

    @_in_order
    def fork(self, seq: int) -> int:
        """A branch with the same positions: it shares the pages until one of the two writes."""
        pages = self._own(seq)
        branch = self._vacant()
        keep = pages[:-(-self._lengths[seq] // self.cache.page)]
        for p in keep:
            self._refs[p] += 1
        self._pages[branch], self._lengths[branch], self._shifts[branch] = list(keep), self._lengths[seq], list(self._shifts[seq])
        self._publish(branch)
        return branch

    @_in_order
    def compact(self, seq: int, keep) -> None:
        """Keeps the given places (ascending) and packs them; the others are forgotten.  Keys stay turned as they are, and the sequence goes on
        behind its last one (``shift_of``).  Forgetting an end moves nothing; else the places go to free pages, or where these do not suffice
        to the front of the sequence's own, as far as no branch shares them."""
        pages, size = self._own(seq), self.cache.page
        keep = [int(p) for p in keep]
        if any(a >= b for a, b in zip(keep, keep[1:])) or (keep and (keep[0] < 0 or keep[-1] >= self._lengths[seq])):
            _refuse("positions to keep are ascending and among the sequence's own")
        n = len(keep)
        if n == 0 or keep[-1] == n - 1:                                                  # only an end is forgotten: nothing moves
            left = pages[:-(-n // size)]
            self._drop(pages[len(left):])
        else:
            same = 0                                                                     # pages at the front that stay as they are
            while (same + 1) * size <= n and keep[(same + 1) * size - 1] == (same + 1) * size - 1:
                same += 1
            need = -(-n // size) - same
            own = set() if need <= len(self._free) else {j for j in range(same, same + need) if self._refs[pages[j]] == 1}
            new = iter(self._take(need - len(own)))
            left = pages[:same] + [pages[j] if j in own else next(new) for j in range(same, same + need)]
            self._move_rows(pages, left, keep, same * size)
            self._drop([p for j, p in enumerate(pages) if j >= same and j not in own])
        self._pages[seq], self._lengths[seq], self._shifts[seq] = left, n, _shifted(self._shifts[seq], keep)
        self._publish(seq)

    def _move_rows(self, pages: list, left: list, keep: list, first: int) -> None:
        """Places ``keep[first:]`` of a sequence in ``pages`` become its places first, first + 1, .. in ``left``, where a page may stand that the
        sequence had there before.  Places move to lower ones, so that in their order none is written before it was read.  A call has no
        destination among its sources: it takes as many places as that allows, or goes by way of the free pages where they hold more."""
        size = self.cache.page
        row = lambda table, i: table[i // size] * size + i % size
        moves = [(a, b) for a, b in ((row(pages, p), row(left, i)) for i, p in enumerate(keep[first:], first)) if a != b]
        by, calls, at = [p * size + r for p in self._free[:-(-len(moves) // size)] for r in range(size)], [], 0
        while at < len(moves):
            read, written, end = set(), set(), at
            while end < len(moves) and moves[end][0] not in written and moves[end][1] not in read:
                read.add(moves[end][0])
                written.add(moves[end][1])
                end += 1
            if end < len(moves) and end - at < len(by):
                end = min(at + len(by), len(moves))
                calls.append([(a, c) for (a, _), c in zip(moves[at:end], by)])
                calls.append([(c, b) for (_, b), c in zip(moves[at:end], by)])
            else:
                calls.append(moves[at:end])
            at = end
        src, dst = (self._numbers([m[i] for call in calls for m in call]) for i in (0, 1))
        at = 0
        for call in calls:
            self.cache.copy_rows(src[at:at + len(call)], dst[at:at + len(call)])
            at += len(call)

    @_in_order
    def pack(self) -> int:
        """Moves pages to the lowest numbers; returns how many pages, from the front, are in use."""
        used = sorted(p for p, n in enumerate(self._refs) if n)
        moves = [(p, i) for p, i in zip(reversed([p for p in used if p >= len(used)]), [p for p in range(len(used)) if self._refs[p] == 0])]
        if moves:
            self.cache.copy_pages(self._numbers([a for a, _ in moves]), self._numbers([b for _, b in moves]))
            to = dict(moves)
            for a, b in moves:
                self._refs[b], self._refs[a] = self._refs[a], 0
            for seq, pages in enumerate(self._pages):
                if pages is not None and any(p in to for p in pages):
                    self._pages[seq] = [to.get(p, p) for p in pages]
                    self._publish(seq)
            self._free = list(range(len(used), self.cache.pages))
        return len(used)
