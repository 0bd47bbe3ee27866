"""The quantized Llama decoder with its sequences in one pool of pages: several of them at a time, branches that share what they have in
common, and memory by the tokens that are there instead of by the longest sequence.

Products, norms and the captured decode step are ``LlamaDecoder``'s; a step's or a portion's attention goes through the ``pages`` entries.
The step is captured once, over the row of page numbers and the position of whichever sequence is bound.
"""
from __future__ import annotations

import torch

from . import _lib, ops, paged
from .decoder import LlamaConfig, LlamaDecoder, ModelWeights, SlotDecoder, rotary_scaling


class PagedLlamaDecoder(LlamaDecoder):
    PAGE = 64

    def __init__(self, ctx: ops.GpuContext, cfg: LlamaConfig, weights: ModelWeights, prefill_chunk: int = 2048, *, n_slots: int, pages: int, freq: torch.Tensor | None = None):
        """``pages`` of PAGE positions for all sequences together; ``freq``: the turns per position of each pair (None: of cfg.rope_theta)."""
        self.n_slots, self._n_pages = n_slots, pages
        freq = paged.rope_frequencies(cfg.head_dim, cfg.rope_theta) if freq is None else freq
        self.rope = paged.Rope(freq.to(torch.device("cuda", ctx.device)))
        super().__init__(ctx, cfg, weights, prefill_chunk)
        self.fused_attention = False
        i32 = dict(dtype=torch.int32, device=self.dev)
        self._q1 = torch.zeros((1, cfg.q_rows), dtype=torch.float32, device=self.dev)
        # of the bound sequence: its pages; its length and the position that the newest token is turned by, pos + (1, shift)
        self._row, self._at, self._plus = torch.full((1, self.pages.table.shape[1]), -1, **i32), torch.zeros(2, **i32), torch.tensor([1, 0], **i32)
        self._len, self._turn = self._at[:1], self._at[1:]
        self._state = torch.zeros((n_slots, 2), **i32)                                                         # position and next token of the others
        self._slot, self._portion, self._turns = None, None, None
        self._done = torch.cuda.Event()
        self._one = self._batch(1, cfg.max_seq)
        self._one.scratch(self.cache.structs[0], cfg.n_heads, 0, 0)                           # (before any capture)

    @classmethod
    def from_gguf(cls, ctx: ops.GpuContext, path, max_seq: int = 32768, prefill_chunk: int = 2048, *, n_slots: int = 4, pages: int | None = None) -> "PagedLlamaDecoder":
        """As ``LlamaDecoder.from_gguf``, with the turns scaled where the file says so (``rope_freqs.weight``: a divisor for each pair;
        ``rope.scaling.factor`` of linear scaling); other scalings are refused.  ``pages`` None: room for every sequence at its longest."""
        turns = {}

        def scaled(kind, linear, factors):
            if kind not in ("none", "linear"):
                raise ops.Hf2qError(_lib.ERR_INVALID_ARGUMENT, f"rotary turns scaled by '{kind}' are not served (have: linear, a divisor for each pair)")
            turns.update(linear=linear, factors=factors)

        def make(ctx, cfg, weights, prefill_chunk):
            factors = turns["factors"]
            freq = paged.rope_frequencies(cfg.head_dim, cfg.rope_theta, linear=turns["linear"])
            if factors is not None:
                freq = (freq.double() / torch.from_numpy(factors).double()).float()
            return cls(ctx, cfg, weights, prefill_chunk, n_slots=n_slots, pages=n_slots * -(-max_seq // cls.PAGE) if pages is None else pages, freq=freq)

        return cls._load_gguf(ctx, path, max_seq, prefill_chunk, make, scaled)

    def _allocate_cache(self) -> None:
        c = self.cfg
        self.cache = paged.PagedCache.allocate(self.ctx, c.n_layers, self._n_pages, self.PAGE, c.n_kv_heads, c.head_dim, torch.int8)
        self.pages = paged.PagePool(self.cache, self.n_slots, c.max_seq, self._ordered)

    def _batch(self, m: int, max_length: int) -> paged.PagedBatch:
        """The bound sequence's last m tokens."""
        start = torch.zeros(2, dtype=torch.int32, device=self.dev)
        start[1:].fill_(m)
        return paged.PagedBatch(self.ctx, start, self._len, self._row, rows=m, max_new=m, max_length=max_length)

    _ordered = SlotDecoder._ordered         # calls on different streams follow one another

    # ---- sequences ------------------------------------------------------------------------------
    def open_slot(self) -> int:
        with self._ordered():
            slot = self.pages.open()
            self._state[slot].zero_()
        return slot

    def close_slot(self, slot: int) -> None:
        with self._ordered():
            self.pages.close(slot)
        if slot == self._slot:
            self._slot = None

    def fork(self, slot: int) -> int:
        """A branch of the sequence as it stands: the tokens so far are shared, what comes next is its own."""
        with self._ordered():
            branch = self.pages.fork(slot)
            self._state[branch] = torch.cat([self.pos, self.tok]) if slot == self._slot else self._state[slot]
        return branch

    def fits(self, lengths) -> bool:
        """The free pages hold new sequences of these lengths, all at once."""
        return sum(-(-n // self.PAGE) for n in lengths) <= self.pages.n_free_pages

    def compact(self, slot: int, keep) -> None:
        """Keeps the given places of the sequence (ascending); the others are forgotten, and it goes on behind the last one."""
        self.pages.compact(slot, keep)

    def pack(self) -> int:
        """Moves the sequences to the pool's lowest pages; returns how many are in use."""
        return self.pages.pack()

    def bind(self, slot: int) -> None:
        self.pages.length_of(slot)                                                       # (raises for a slot that is not in use)
        if slot == self._slot:
            return
        with self._ordered():
            if self._slot is not None:
                self._state[self._slot] = torch.cat([self.pos, self.tok])
            self.pos.copy_(self._state[slot, :1])
            self.tok.copy_(self._state[slot, 1:])
            self._row.copy_(self.pages.table[slot:slot + 1])
        self._slot = slot

    def _reserve(self, n: int) -> None:
        if self._slot is None:
            raise RuntimeError("no sequence is bound")
        self.pages.reserve(self._slot, n)
        self._row.copy_(self.pages.table[self._slot:self._slot + 1])
        self._plus[1:].fill_(self.pages.shift_of(self._slot))                            # (the pool may have compacted the sequence)

    def extend(self, slot: int, ids: torch.Tensor, want) -> torch.Tensor:
        self.bind(slot)
        out = torch.empty((len(want), self.cfg.vocab), dtype=torch.float32, device=self.dev)
        self.prefill(ids, start=self.pages.length_of(slot), want=list(want), want_out=out)
        return out

    def prefill(self, ids: torch.Tensor, start: int = 0, want=(), want_out=None) -> None:
        """As ``LlamaDecoder.prefill`` for the bound sequence; ``start`` is its length."""
        n = int(ids.numel())
        if self._slot is None or start != self.pages.length_of(self._slot):
            raise ops.Hf2qError(_lib.ERR_INVALID_ARGUMENT, "a portion starts where the bound sequence ends")
        if n == 0 or start + n >= self.cfg.max_seq:
            raise ops.Hf2qError(_lib.ERR_INVALID_ARGUMENT, f"sequence length {start + n} must be in 1..max_seq-1 and grow")
        with self._ordered():
            self._reserve(n)
            super().prefill(ids, start, want, want_out)
            self.pages.advance(self._slot, n)
            self._portion = self._q = self._turns = None

    def generate(self, n: int, use_graph: bool = True, collect: bool = True):
        """As ``LlamaDecoder.generate`` for the bound sequence."""
        if n < 1:
            return torch.empty(0, dtype=torch.int32, device=self.dev) if collect else None
        with self._ordered():
            self._reserve(n)
            self.pos.fill_(self.pages.length_of(self._slot))
            out = super().generate(n, use_graph, collect)
            self.pages.advance(self._slot, n)
        return out

    def _prefill_buffers(self, m, panels):
        """As ``LlamaDecoder``'s; a stream that one call has used them on may still be at work when another call, on another stream, replaces them
        by larger ones."""
        have = super()._prefill_buffers(m, panels)
        for t in have.values():
            if isinstance(t, torch.Tensor):
                t.record_stream(torch.cuda.current_stream(self.dev))
        return have

    # ---- attention ------------------------------------------------------------------------------
    def decode_step(self) -> None:
        torch.add(self.pos, self._plus, out=self._at)
        super().decode_step()

    @property
    def launches_per_token(self) -> int:
        """At most: over caches of a few pages attention has no parts to join."""
        return super().launches_per_token + 1

    def _attend_step(self, i: int) -> None:
        c = self.cfg
        self.cache.append(i, self._one, self.rope, self.qkv, c.n_heads, self._q1, positions=self._turn)
        self.cache.attend(i, self._one, self._q1, c.n_heads, self.att)

    def _attend_portion(self, i: int, qkv, m: int, p0: int, att) -> None:
        c = self.cfg
        if i == 0:
            self._len.fill_(p0 + m)
            self._portion, self._q = self._batch(m, p0 + m), torch.empty((m, c.q_rows), dtype=torch.float32, device=self.dev)
            shift = self.pages.shift_of(self._slot)
            self._turns = torch.arange(p0 + shift, p0 + shift + m, dtype=torch.int32, device=self.dev) if shift else None
        self.cache.append(i, self._portion, self.rope, qkv, c.n_heads, self._q, positions=self._turns)
        self.cache.attend(i, self._portion, self._q, c.n_heads, att)
