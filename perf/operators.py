"""Operators of a paged key-value cache: what is timed, and their plain forms.

A cache of a layer keeps keys and values in pages [pages, kv_heads, page, dim], bf16 or signed bytes with one f32 scale per (head,
position).  A batch names sequences by a row of page numbers each, how many positions each holds, and which of the call's rows are its
newest tokens.  Four kinds of case:

  append   rotary turn of queries and keys (pairs side by side or in halves, all of the head or its first part, any table of
           frequencies), keys and values into the pages
  attend   the newest tokens of every sequence over its pages, causal, with a window and first positions that stay visible or without
  copy     whole pages of all layers (a sequence that forks, a pool that is packed)
  compact  single positions of all layers (a sequence of which some positions are kept)

Lengths differ from sequence to sequence by a rule on the case's numbers; values come from the seed.
"""
import math
import zlib

import torch

own = False
DEV = "cuda"
_CTX = None


# ---- the cases --------------------------------------------------------------------------------------
def listed():
    llama = {"heads": 32, "kv_heads": 8, "dim": 128}
    return [
        # one more token of each of 16 sequences: the rows a decode step writes
        {"name": "append-step", "kind": "append", "cache": "bf16", "seqs": 16, "new": 1, "context": 2048, "spread": 0.8, **llama, "page": 16, "x": "f32",
         "rot": 128, "halves": False, "scaling": "none"},
        # portions of three prompts, half of each head turned, frequencies stretched for long contexts
        {"name": "append-prompt", "kind": "append", "cache": "int8", "seqs": 3, "new": 2048, "context": 0, "spread": 0.6, **llama, "page": 32, "x": "f32",
         "rot": 64, "halves": True, "scaling": "bands"},
        # the smallest attention: one sequence, one token, a short context
        {"name": "step-short", "kind": "attend", "cache": "bf16", "seqs": 1, "new": 1, "context": 200, "spread": 0.0, **llama, "page": 16, "window": 0,
         "sinks": 0, "out": "bf16"},
        # a decode step of 32 sequences of all lengths
        {"name": "step-32-sequences", "kind": "attend", "cache": "int8", "seqs": 32, "new": 1, "context": 8191, "spread": 0.9, **llama, "page": 16, "window": 0,
         "sinks": 0, "out": "bf16"},
        # one token behind a very long context
        {"name": "step-long", "kind": "attend", "cache": "int8", "seqs": 1, "new": 1, "context": 131071, "spread": 0.0, **llama, "page": 64, "window": 0,
         "sinks": 0, "out": "f16"},
        # a decode step that streams: a window and four first positions, heads in groups of five
        {"name": "step-window", "kind": "attend", "cache": "bf16", "seqs": 24, "new": 1, "context": 20000, "spread": 0.7, "heads": 40, "kv_heads": 8, "dim": 64,
         "page": 16, "window": 1024, "sinks": 4, "out": "bf16"},
        # drafted tokens of eight sequences, checked at once, heads in groups of seven
        {"name": "drafts", "kind": "attend", "cache": "bf16", "seqs": 8, "new": 5, "context": 3001, "spread": 0.5, "heads": 28, "kv_heads": 4, "dim": 128,
         "page": 32, "window": 0, "sinks": 0, "out": "bf16"},
        # a small portion of a prompt behind a long context
        {"name": "chunk-long", "kind": "attend", "cache": "int8", "seqs": 1, "new": 64, "context": 32768, "spread": 0.0, **llama, "page": 64, "window": 0,
         "sinks": 0, "out": "f16"},
        # portions of six prompts of odd lengths, windowed
        {"name": "chunks-window", "kind": "attend", "cache": "bf16", "seqs": 6, "new": 701, "context": 6007, "spread": 0.8, **llama, "page": 16, "window": 2048,
         "sinks": 16, "out": "bf16"},
        # a large portion of a long prompt
        {"name": "prompt", "kind": "attend", "cache": "int8", "seqs": 1, "new": 4096, "context": 12288, "spread": 0.0, **llama, "page": 64, "window": 0,
         "sinks": 0, "out": "f16"},
        # a sequence forks: its last, partly filled page is copied for every branch, in all layers
        {"name": "fork", "kind": "copy", "cache": "int8", "layers": 32, "pages": 96, "moved": 12, "kv_heads": 8, "dim": 128, "page": 16},
        # half of a long sequence's positions are kept and packed into other pages
        {"name": "compact", "kind": "compact", "cache": "bf16", "layers": 4, "rows": 16384, "kept": 8192, "kv_heads": 8, "dim": 128, "page": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


MOST_PAIRS = 32 * 4096 * 14336                   # (head, query, key) triples of the largest listed case
MOST_SCORES = 32 * 4096 * 16384                  # scores that the plain form keeps for it


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "attend", "copy", "compact"])
    kv_heads, group = rng.randint(1, 12), rng.randint(1, 12)
    shape = {"heads": kv_heads * group, "kv_heads": kv_heads, "dim": rng.choice([64, 128])}
    cache, page = rng.choice(["bf16", "int8"]), rng.choice([16, 32, 64, 128])
    if kind == "append":
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 2048)
        return {"kind": kind, "cache": cache, "seqs": _log(rng, 1, 32 if new == 1 else 4), "new": new, "context": rng.randint(0, 500),
                "spread": round(rng.uniform(0, 0.9), 2), **shape, "page": page, "x": rng.choice(["f32", "bf16"]), "rot": rng.choice([shape["dim"], 32, 8 * rng.randint(1, 7)]),
                "halves": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "bands"])}
    if kind == "copy":
        layers, moved = rng.randint(1, 32), _log(rng, 1, 256)
        return {"kind": kind, "cache": cache, "layers": layers, "pages": 2 * moved + rng.randint(0, 64), "moved": moved, "kv_heads": kv_heads, "dim": shape["dim"], "page": page}
    if kind == "compact":
        rows = _log(rng, 2, 8192)
        return {"kind": kind, "cache": cache, "layers": rng.randint(1, 4), "rows": rows, "kept": rng.randint(1, rows), "kv_heads": kv_heads, "dim": shape["dim"], "page": page}
    while True:
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
        case = {"kind": kind, "cache": cache, "seqs": _log(rng, 1, 48), "new": new, "context": _log(rng, 1, 65536), "spread": round(rng.uniform(0, 0.9), 2), **shape,
                "page": page, "window": 0 if rng.random() < 0.6 else _log(rng, 16, 8192), "sinks": rng.choice([0, 0, 1, 4, 70]),
                "out": rng.choice(["bf16", "f16"]) if cache == "int8" else "bf16"}        # (a quantized decoder's next product takes f16, a bf16 design's bf16)
        longest = case["context"] + new
        if case["seqs"] * case["heads"] * new * longest <= MOST_SCORES // 2 and case["seqs"] * longest * kv_heads <= 1 << 22 and \
                case["seqs"] * case["heads"] * new * longest <= MOST_PAIRS // 2:
            return case


def _lengths(case):
    """(new tokens, positions before them) of every sequence."""
    out = []
    for i in range(case["seqs"]):
        a, b = (0.618034 * i) % 1.0, (0.381966 * i * i) % 1.0
        new = case["new"] if case["new"] == 1 else max(1, round(case["new"] * (1 - case["spread"] * a)))
        out.append((new, round(case["context"] * (1 - case["spread"] * b))))
    return out


# ---- inputs -----------------------------------------------------------------------------------------
def _generator(seed, *tag):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr((int(seed),) + tag).encode()))


def _cache(case, layers, pages, g):
    """Pages full of earlier tokens (a free page holds what was there before)."""
    shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
    out = {}
    for name in ("k", "v"):
        values = torch.randn(shape, generator=g, device=DEV)
        if case["cache"] == "int8":
            scale = values.abs().amax(dim=-1) / 127
            out[name], out[name + "_scale"] = torch.round(values / scale[..., None]).to(torch.int8), scale
        else:
            out[name], out[name + "_scale"] = values.to(torch.bfloat16), None
    return out


def frequencies(rot, scaling, theta=500000.0):
    """Turns (radians) per position of each pair: theta^(-2i/rot); "linear": a quarter of that; "bands": long wavelengths divided by 8, short ones
    kept, those between in proportion, for a model made for 8192 positions."""
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling == "linear":
        f = f / 4
    if scaling == "bands":
        part = ((8192 * f / (2 * math.pi) - 1) / 3).clamp(0, 1)
        f = f / 8 * (1 - part) + f * part
    return f.to(torch.float32)


def prepare(case, seed):
    g = _generator(seed, tuple(sorted((k, v) for k, v in case.items() if k != "name")))
    cpu = torch.Generator().manual_seed(zlib.crc32(repr((int(seed), "order")).encode()))
    i32 = dict(dtype=torch.int32, device=DEV)
    if case["kind"] == "copy":
        order = torch.randperm(case["pages"], generator=cpu)
        return {"case": case, **_cache(case, case["layers"], case["pages"], g), "src": order[:case["moved"]].to(**i32), "dst": order[case["moved"]:2 * case["moved"]].to(**i32)}
    if case["kind"] == "compact":
        old, kept = -(-case["rows"] // case["page"]), case["kept"]
        order = torch.randperm(old + -(-kept // case["page"]), generator=cpu)
        rows = (order[:, None] * case["page"] + torch.arange(case["page"])[None]).reshape(-1)      # position of a sequence -> row of the cache
        src = torch.sort(torch.randperm(case["rows"], generator=cpu)[:kept]).values
        return {"case": case, **_cache(case, case["layers"], len(order), g), "src": rows[src].to(**i32), "dst": rows[old * case["page"]:][:kept].to(**i32)}
    lengths = _lengths(case)
    total = [n + c for n, c in lengths]
    pages = [-(-t // case["page"]) for t in total]
    order, table, at = torch.randperm(sum(pages) + 3, generator=cpu), torch.zeros((case["seqs"], max(pages)), dtype=torch.int32), 0
    for s, n in enumerate(pages):
        table[s, :n] = order[at:at + n]
        at += n
    start = torch.cumsum(torch.tensor([0] + [n for n, _ in lengths]), 0)
    rows, width = int(start[-1]), case["heads"] * case["dim"]
    st = {"case": case, **_cache(case, 1, len(order), g), "start": start.to(**i32), "length": torch.tensor(total).to(**i32), "table": table.to(**i32), "rows": rows,
          "most_new": max(n for n, _ in lengths), "longest": max(total)}
    if case["kind"] == "append":
        st["x"] = torch.randn((rows, width + 2 * case["kv_heads"] * case["dim"]), generator=g, device=DEV).to(torch.bfloat16 if case["x"] == "bf16" else torch.float32)
        st["freq"] = frequencies(case["rot"], case["scaling"]).to(DEV)
        st["q"] = torch.empty((rows, width), dtype=torch.float32, device=DEV)
        st["values"] = [torch.empty(st["k"].shape, dtype=torch.bfloat16, device=DEV) for _ in "kv"] if case["cache"] == "int8" else None
    else:
        st["q"] = torch.randn((rows, width), generator=g, device=DEV).to(torch.bfloat16)
        st["o"] = torch.empty((rows, width), dtype=torch.bfloat16 if case["out"] == "bf16" else torch.float16, device=DEV)
    return st


# ---- one pass ---------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        _own(state, case)
    else:
        {"append": _append, "attend": _attend, "copy": _copy, "compact": _compact}[case["kind"]](state, case)
    if case["kind"] == "attend":
        return {"out": state["o"]}
    if case["kind"] == "append":
        out = {"q": state["q"]}
        if case["cache"] == "int8":              # bytes come back as the values they stand for
            out["k"], out["v"] = (torch.mul(state[n], state[n + "_scale"][..., None], out=t) for n, t in zip("kv", state["values"]))
            return out
        return {**out, "k": state["k"], "v": state["v"]}
    return {n: state[n] for n in ("k", "v", "k_scale", "v_scale") if state[n] is not None}


def _own(st, case):
    global _CTX
    if "cache" not in st:                        # what a program keeps: one context, the cache, the step's batch, the turns of the model
        from hf2q_b200 import ops, paged
        if _CTX is None:
            _CTX = ops.GpuContext(0)
        st["cache"] = paged.PagedCache(_CTX, st["k"], st["v"], st["k_scale"], st["v_scale"])
        if "table" in st:
            st["batch"] = paged.PagedBatch(_CTX, st["start"], st["length"], st["table"], rows=st["rows"], max_new=st["most_new"], max_length=st["longest"])
        if "freq" in st:
            st["rope"] = paged.Rope(st["freq"], halves=case["halves"])
    cache = st["cache"]
    if case["kind"] == "append":
        cache.append(0, st["batch"], st["rope"], st["x"], case["heads"], st["q"])
    elif case["kind"] == "attend":
        cache.attend(0, st["batch"], st["q"], case["heads"], st["o"], window=case["window"], sinks=case["sinks"])
    elif case["kind"] == "copy":
        cache.copy_pages(st["src"], st["dst"])
    else:
        cache.copy_rows(st["src"], st["dst"])


# ---- plain forms ------------------------------------------------------------------------------------
def _places(st, page):
    """Sequence, position, page and row in the page of every new token."""
    t = torch.arange(st["rows"], device=DEV)
    seq = torch.searchsorted(st["start"], t.to(torch.int32), right=True) - 1
    pos = st["length"][seq].long() - st["start"][seq + 1].long() + t
    return seq, pos, st["table"][seq, pos // page].long(), pos % page


def _append(st, case):
    h, kv, d, rot = case["heads"], case["kv_heads"], case["dim"], case["rot"]
    _, pos, page, row = _places(st, case["page"])
    x = st["x"].float().view(st["rows"], h + 2 * kv, d)
    angle = pos.double()[:, None] * st["freq"].double()[None]        # (far positions need more than 32 bits)
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    turned, qk = x.clone(), x[:, :h + kv]
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if case["halves"] else (slice(0, rot, 2), slice(1, rot, 2))
    a, b = qk[..., first], qk[..., second]
    turned[:, :h + kv, first] = a * c - b * s
    turned[:, :h + kv, second] = a * s + b * c
    st["q"].copy_(turned[:, :h].reshape(st["rows"], h * d))
    _store(st, "k", turned[:, h:h + kv], page, row)
    _store(st, "v", turned[:, h + kv:], page, row)


def _store(st, name, values, page, row):
    if st[name + "_scale"] is None:
        st[name][0, page, :, row] = values.to(torch.bfloat16)
        return
    top = values.abs().amax(dim=-1)
    limit = torch.full_like(top, 127.0)
    st[name][0, page, :, row] = torch.round(values * torch.where(top > 0, limit / top, torch.zeros_like(top))[..., None]).to(torch.int8)
    st[name + "_scale"][0, page, :, row] = top / limit


def _attend(st, case):
    h, kv, d, size = case["heads"], case["kv_heads"], case["dim"], case["page"]
    seqs, most = case["seqs"], st["most_new"]
    seq, pos, _, _ = _places(st, size)
    place = torch.arange(st["rows"], device=DEV) - st["start"][seq].long()
    q = torch.zeros((seqs, most, kv, h // kv, d), device=DEV)
    q[seq, place] = st["q"].float().view(-1, kv, h // kv, d)
    at = torch.zeros((seqs, most), dtype=torch.long, device=DEV)
    at[seq, place] = pos

    def gathered(name):
        t = st[name][0][st["table"].long()].float()                                     # [seqs, pages, kv, size, d]
        if st[name + "_scale"] is not None:
            t = t * st[name + "_scale"][0][st["table"].long()][..., None]
        return t.transpose(1, 2).reshape(seqs, kv, -1, d)

    k, v = gathered("k"), gathered("v")
    j = torch.arange(k.shape[2], device=DEV)
    seen = j <= at[..., None]
    if case["window"]:
        seen &= (at[..., None] - j < case["window"]) | (j < case["sinks"])
    s = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, d), k.transpose(2, 3)).view(seqs, kv, h // kv, most, -1)
    s = (s * (1 / math.sqrt(d))).masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    o = torch.matmul(p.view(seqs, kv, -1, p.shape[-1]), v).view(seqs, kv, h // kv, most, d) / p.sum(dim=-1, keepdim=True)
    st["o"].copy_(o.permute(0, 3, 1, 2, 4)[seq, place].reshape(st["rows"], h * d))


def _arrays(st):
    return [st[n] for n in ("k", "v", "k_scale", "v_scale") if st[n] is not None]


def _copy(st, case):
    src, dst = st["src"].long(), st["dst"].long()
    _ = [t.index_copy_(1, dst, t.index_select(1, src)) for t in _arrays(st)]


def _compact(st, case):
    src, dst, size = st["src"].long(), st["dst"].long(), case["page"]
    for t in _arrays(st):
        t[:, dst // size, :, dst % size] = t[:, src // size, :, src % size]


# ---- what a pass cannot do without ------------------------------------------------------------------
def _pairs(first, count, window, sinks):
    """(query, key) pairs of `count` queries from position `first` on, and the keys that any of them sees."""
    if not window:
        return count * first + count * (count + 1) // 2, first + count
    pairs = 0
    for p in range(first, first + count):
        low = max(0, p - window + 1)
        pairs += p + 1 - low + min(sinks, low)
    low = max(0, first - window + 1)
    return pairs, first + count - low + min(sinks, low)


def work(case):
    d, kv, byte = case["dim"], case["kv_heads"], case["cache"] == "int8"
    row = 2 * kv * (d + 4 if byte else 2 * d)                                           # key and value of a position
    if case["kind"] == "copy":
        return {"bytes": 2 * case["layers"] * case["moved"] * case["page"] * row + 8 * case["moved"], "flops": 0}
    if case["kind"] == "compact":
        return {"bytes": 2 * case["layers"] * case["kept"] * row + 8 * case["kept"], "flops": 0}
    lengths = _lengths(case)
    rows = sum(n for n, _ in lengths)
    if case["kind"] == "append":
        x = (case["heads"] + 2 * kv) * d * (2 if case["x"] == "bf16" else 4)
        return {"bytes": rows * (x + 4 * case["heads"] * d + row), "flops": rows * (3 * (case["heads"] + kv) * case["rot"] + (6 * kv * d if byte else 0))}
    each = [_pairs(c, n, case["window"], case["sinks"]) for n, c in lengths]
    return {"bytes": sum(keys for _, keys in each) * row + rows * case["heads"] * d * 4, "flops": 4 * d * case["heads"] * sum(p for p, _ in each)}


# ---- the same in 64 bits ----------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] in ("copy", "compact"):
        size = case["page"] if case["kind"] == "compact" else 1
        out = {}
        for name in ("k", "v", "k_scale", "v_scale"):
            if st[name] is None:
                continue
            if not st[name].is_floating_point():
                out[name] = None
                continue
            t = st[name].transpose(1, 2) if size == 1 else st[name].transpose(1, 2).flatten(2, 3)      # [layers, kv, pages or positions, ..]
            for n in range(0, len(st["src"]), 4096):
                t[:, :, st["dst"][n:n + 4096].long()] = t[:, :, st["src"][n:n + 4096].long()]
            shape = st[name].shape
            out[name] = (t if size == 1 else t.unflatten(2, (shape[1], size))).transpose(1, 2).double()
        return out
    h, kv, d, size = case["heads"], case["kv_heads"], case["dim"], case["page"]
    start, table = st["start"].tolist(), st["table"].long()
    if case["kind"] == "append":
        q = torch.empty((st["rows"], h, d), dtype=torch.float64, device=DEV)
        values = {n: st[n][0].double() * (1 if st[n + "_scale"] is None else st[n + "_scale"][0].double()[..., None]) for n in "kv"}
        w = case["rot"] // 2
        for s, total in enumerate(st["length"].tolist()):
            a, b = start[s], start[s + 1]
            x = st["x"][a:b].double().view(b - a, -1, d).clone()
            p = torch.arange(total - (b - a), total, device=DEV)
            phase = torch.polar(torch.ones((b - a, w), dtype=torch.float64, device=DEV), p.double().outer(st["freq"].double()))[:, None]
            part = x[:, :h + kv, :2 * w]
            z = torch.complex(*part.unflatten(2, (2, w)).unbind(2)) if case["halves"] else torch.view_as_complex(part.unflatten(2, (w, 2)).contiguous())
            z = torch.view_as_real(z * phase)
            x[:, :h + kv, :2 * w] = (z.transpose(2, 3) if case["halves"] else z).flatten(2)
            q[a:b] = x[:, :h]
            for n, t in (("k", x[:, h:h + kv]), ("v", x[:, h + kv:])):
                if case["cache"] == "int8":
                    unit = t.abs().amax(-1, keepdim=True) / 127
                    t = torch.round(t / unit) * unit
                values[n][table[s, p // size], :, p % size] = t
        return {"q": q.view(st["rows"], -1), "k": values["k"][None], "v": values["v"][None]}
    out = torch.empty((st["rows"], h, d), dtype=torch.float64, device=DEV)
    for s, total in enumerate(st["length"].tolist()):
        a, b = start[s], start[s + 1]
        own_pages = table[s, :-(-total // size)]
        for head in range(kv):
            k, v = (st[n][0, own_pages, head].double() * (1 if st[n + "_scale"] is None else st[n + "_scale"][0, own_pages, head].double()[..., None]) for n in "kv")
            k, v = k.reshape(-1, d)[:total], v.reshape(-1, d)[:total]
            for t0 in range(a, b, 512):
                t1 = min(t0 + 512, b)
                q = st["q"][t0:t1].double().view(t1 - t0, kv, -1, d)[:, head]
                gap = torch.arange(total - (b - t0), total - (b - t1), device=DEV)[:, None] - torch.arange(total, device=DEV)
                hidden = gap < 0
                if case["window"]:
                    hidden |= (gap >= case["window"]) & (torch.arange(total, device=DEV) >= case["sinks"])
                logits = torch.einsum("qgd,jd->qgj", q, k) / math.sqrt(d)
                logits[hidden[:, None].expand_as(logits)] = -math.inf
                out[t0:t1].view(t1 - t0, kv, -1, d)[:, head] = torch.einsum("qgj,jd->qgd", torch.softmax(logits, -1), v)
    return {"out": out.view(st["rows"], -1)}
