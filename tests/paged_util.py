"""A paged cache with known contents, attention and append over it in 64 bits, and how far a result in fewer bits may be off."""
import math

import torch

STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # largest rounding, relative to the value


class Pages:
    """Sequences of ``lengths`` = [(new, before)] in pages that lie in random order; rows of pages that hold no position are poisoned."""

    def __init__(self, lengths, kv_heads, group, dim, page, dtype, seed, layers=1, spare=2, scale=1.0, ld_extra=0):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.kv_heads, self.group, self.dim, self.page, self.dtype = lengths, kv_heads, group, dim, page, dtype
        self.heads, self.rows, self.layers = kv_heads * group, sum(n for n, _ in lengths), layers
        total = [n + c for n, c in lengths]
        need = [-(-t // page) for t in total]
        order = torch.randperm(sum(need) + spare, generator=g)
        self.n_pages = len(order)
        self.table = torch.full((len(lengths), max(need + [1]) + ld_extra), 1 << 30, dtype=torch.int32)          # (past the length nothing may be read)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.start = torch.cumsum(torch.tensor([0] + [n for n, _ in lengths]), 0).to(torch.int32)
        self.length = torch.tensor(total, dtype=torch.int32)
        shape = (layers, self.n_pages, kv_heads, page, dim)
        used = torch.zeros((self.n_pages, page), dtype=torch.bool)
        for s, t in enumerate(total):
            p = torch.arange(t)
            used[self.table[s, p // page].long(), p % page] = True
        self.used = used[None, :, None].expand(shape[:4])
        self.k, self.v, self.k_scale, self.v_scale = None, None, None, None
        for name in "kv":
            x = torch.randn(shape, generator=g) * scale
            if dtype == torch.int8:
                s = x.abs().amax(-1) / 127
                setattr(self, name, torch.where(self.used[..., None], torch.round(x / s[..., None]), torch.tensor(-128.0)).to(torch.int8))
                setattr(self, name + "_scale", torch.where(self.used, s, torch.tensor(math.nan)))
            else:
                setattr(self, name, torch.where(self.used[..., None], x, torch.tensor(math.nan)).to(dtype))
        self.q = torch.randn((self.rows, self.heads * dim), generator=g)
        self.x = torch.randn((self.rows, (self.heads + 2 * kv_heads) * dim), generator=g)

    def cache(self, ctx):
        from hf2q_b200 import paged
        dev = lambda t: None if t is None else t.cuda()
        return paged.PagedCache(ctx, dev(self.k), dev(self.v), dev(self.k_scale), dev(self.v_scale))

    def batch(self, ctx, max_new=None, max_length=None, rows=None):
        from hf2q_b200 import paged
        return paged.PagedBatch(ctx, self.start.cuda(), self.length.cuda(), self.table.cuda(), rows=self.rows if rows is None else rows,
                                max_new=max(n for n, _ in self.lengths) if max_new is None else max_new, max_length=int(self.length.max()) if max_length is None else max_length)

    def values(self, name, s, layer=0):
        """Keys or values of a sequence [kv_heads, positions, dim] in 64 bits."""
        p = torch.arange(int(self.length[s]))
        page, row = self.table[s, p // self.page].long(), p % self.page
        t = getattr(self, name)[layer, page, :, row].double()
        scale = getattr(self, name + "_scale")
        return (t if scale is None else t * scale[layer, page, :, row].double()[..., None]).transpose(0, 1)


def attention(c: Pages, q, q_dtype, out_dtype, scale=None, window=0, sinks=0):
    """(result, largest error) of every element.  With u the largest rounding of the type that the products take (f16 for codes, bf16 for
    bf16 pages): a score s is off by at most e = scale sum |q| |k| (u_q + (dim + 8) 2^-24), u_q = u unless q is exact in that type,
    so each weight by a factor of 1 +- 2 e, above and below the fraction; each weight above it is rounded once more, by u.  Sums of n terms
    in 32 bits and the exponentials add (n / 16 + 64) 2^-24 (terms of a block are added in a tree or in the tensor core), the result's
    rounding its own step.  Codes: weights below the f16 normal range are off by at most 2^-36 of the largest value scale each."""
    scale = c.dim ** -0.5 if scale is None else scale
    out, tol = torch.zeros((c.rows, c.heads, c.dim), dtype=torch.float64), torch.zeros((c.rows, c.heads, c.dim), dtype=torch.float64)
    qd = q.to(q_dtype).double().view(c.rows, c.kv_heads, c.group, c.dim)
    work = torch.float16 if c.dtype == torch.int8 else torch.bfloat16
    u = STEP[work]
    exact = q_dtype == torch.bfloat16
    for s, total in enumerate(c.length.tolist()):
        a, b = int(c.start[s]), int(c.start[s + 1])
        if a == b:
            continue
        k, v = c.values("k", s), c.values("v", s)
        i, j = torch.arange(total - (b - a), total)[:, None], torch.arange(total)[None]
        seen = (j <= i) & (((i - j < window) | (j < sinks)) if window else True)
        x = torch.einsum("rhgd,hjd->rhgj", qd[a:b], k) * scale
        size = torch.einsum("rhgd,hjd->rhgj", qd[a:b].abs(), k.abs()) * abs(scale)
        hide = ~seen[:, None, None].expand_as(x)
        x = x.masked_fill(hide, -math.inf)
        e = size.masked_fill(hide, 0).amax(-1) * ((0 if exact else u) + (c.dim + 8) * 2.0 ** -24)
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(top.isinf(), 0.0, top))
        p = p.masked_fill(hide, 0)
        l = p.sum(-1, keepdim=True)
        p = torch.where(l > 0, p / torch.where(l > 0, l, 1.0), 0.0)
        o = torch.einsum("rhgj,hjd->rhgd", p, v)
        spread = torch.einsum("rhgj,hjd->rhgd", p, v.abs())
        out[a:b] = o.reshape(b - a, c.heads, c.dim)
        t = spread * (u + 4 * e[..., None] + (total / 16 + 64) * 2.0 ** -24) + STEP[out_dtype] * o.abs() * 1.01 + 2.0 ** -25 * (out_dtype == torch.float16)
        if c.dtype == torch.int8:
            t = t + total * 127 * c.v_scale.nan_to_num(0).max().double() * 2.0 ** -36
        tol[a:b] = t.reshape(b - a, c.heads, c.dim)
    return out.view(c.rows, -1), tol.view(c.rows, -1)


def close(got, want, tol, what=""):
    d = (got.double().cpu() - want).abs()
    worst = (d / tol.clamp(min=1e-300)).max().item() if d.numel() else 0.0
    assert bool((d <= tol).all()), f"{what}: {int((~(d <= tol)).sum())} of {d.numel()} outside, worst {worst:.2f} of what is allowed"
    return worst


def turned(x, pos, freq, rot, halves, factor=1.0):
    """Heads [rows, heads, dim] in 64 bits, turned."""
    x = x.double().clone()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if halves else (slice(0, rot, 2), slice(1, rot, 2))
    angle = pos.double()[:, None] * freq.double()[None]
    c, s = torch.cos(angle)[:, None] * factor, torch.sin(angle)[:, None] * factor
    p, q = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = p * c - q * s, p * s + q * c
    return x
