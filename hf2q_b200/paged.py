"""A key-value cache in pages, for many sequences: ctypes view of the ``pages`` entries of the C ABI and the host side of the pool.

``PagedCache`` holds the pages of one or several layers and launches the entries on torch's current stream; ``PagedBatch`` names the
sequences of a call by arrays on the device; ``Rope`` is a model's rotary turn; ``PagePool`` keeps, on the host, which sequence owns
which page: it hands pages out, shares them between branches of a sequence, and packs and frees them.
"""
from __future__ import annotations

import ctypes as C
import math

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
        if n >= rows and w >= width and (one == 1 or w <= 1) and (ld >= width or rows <= 1):
            return ld if rows > 1 else max(ld, width)
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
        if not 0 <= max_new <= rows or not max_new <= max_length:
            _refuse("max_new is at most rows and at most max_length")
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
        at = lambda t, layer: None if t is None else t[layer].data_ptr()
        self._structs = [_Pages(at(k, i), at(v, i), at(k_scale, i), at(v_scale, i), self.pages, self.page, self.kv_heads, self.dim, DT_I8 if codes else DT_BF16)
                         for i in range(self.layers)]
        self._refs, self._scale = [C.byref(s) for s in self._structs], self.dim ** -0.5
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
        if window < 0 or sinks < 0:
            _refuse("window and sinks are not negative")
        scratch = batch.scratch(self._structs[layer], heads, window, sinks)
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
