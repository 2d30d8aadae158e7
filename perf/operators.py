"""The operators of serving in 4 bits, as measurable cases: Linears over weights of 4 bits with group scales, and a paged
cache whose keys and values are held in 4 bits — storing rows and reading them back, the attention that reads it, and the
bookkeeping of its pages (forking, freeing, growing and compacting sequences).

Weights: W[n, k] = scale[n, k // group]·(value[n, k] − zero[n, k // group]), value 0 … 15, scale and zero bf16 (zero 8 where
none is given); y = x·Wᵀ + bias.
Cache: a row of a head is cut into groups of 64 entries; of a group with least and largest entry lo and hi, scale =
bf16(hi / 15 − lo / 15), middle = bf16(lo + 8·scale), value = clamp(rint((x − middle) / scale), −8, 7) (0 where scale is 0),
and what is read is middle + scale·value.  A sequence's tokens lie in pages of 64 that its row of the table lists; a page is
free while its count of references is 0, and the lowest free page is taken first.
A case is a dict of plain values whose "kind" says which operator it calls.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
PAGE, GROUP = 64, 64


def listed():
    return [
        # the smallest call: one decoded row through the merged q | k | v of a small model, with its bias
        dict(name="linear_one", kind="linear", rows=1, n=1152, k=896, group=64, zero=False, bias=True),
        # one decoded row through the merged gate | up of a large model: the weight stream itself
        dict(name="linear_token", kind="linear", rows=1, n=28672, k=4096, group=128, zero=True, bias=False),
        # a decode batch of eight sequences through a down-projection, finest groups, an odd number of groups
        dict(name="linear_batch", kind="linear", rows=8, n=2048, k=4896, group=32, zero=False, bias=False),
        # a prompt through an out-projection
        dict(name="linear_prompt", kind="linear", rows=512, n=4096, k=4096, group=128, zero=False, bias=False),
        # two short conversations of a small model, seven query heads to a key/value head
        dict(name="attn_short", kind="attention", heads=14, kv_heads=2, dim=64, lengths="23,40", counts="1,1", window=0),
        # one decoded token over a long context
        dict(name="attn_long", kind="attention", heads=24, kv_heads=8, dim=128, lengths="32768", counts="1", window=0),
        # a decode batch of unequal sequences as a server holds them, one of them without pages for its token
        dict(name="attn_batch", kind="attention", heads=16, kv_heads=8, dim=128, counts="1," * 23 + "1", window=0,
             lengths="1,7,63,64,65,130,200,-1,333,512,700,901,1024,1500,1777,2048,2500,2999,3333,4096,5000,6001,7000,8191"),
        # a further piece of a long prompt over what the cache holds of it, beside a token under a window
        dict(name="attn_piece", kind="attention", heads=16, kv_heads=8, dim=128, lengths="4353,1900", counts="257,1", window=1024),
        # the new rows of a decode batch, into the cache and back
        dict(name="store_batch", kind="store", kv_heads=8, dim=128, firsts="0,1,15,63,64,100,250,777,1023,2000,3000,4095", counts="1," * 11 + "1"),
        # a prompt's rows into the cache and back, two sequences, the second behind what it has already
        dict(name="store_prompt", kind="store", kv_heads=8, dim=128, firsts="0,37", counts="2048,1001"),
        # sampling eight answers of one prompt: the last answers' pages are given back, the prompt forked, a token's room made for each
        dict(name="fork", kind="fork", layers=4, kv_heads=2, dim=128, n_pages=384, length=1001, copies=8),
        # half of the sequences leave, the others' pages move together, new ones of their size come; twice, so that all have moved
        dict(name="compact", kind="compact", layers=4, kv_heads=4, dim=128, n_pages=256, lengths="1,64,65,500,1000,2300"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _sizes(rng, n, lo, hi):
    return ",".join(str(_log(rng, lo, hi)) for _ in range(n))


def draw(rng):
    kind = rng.choice(["linear", "linear", "attention", "attention", "store", "fork", "compact"])
    if kind == "linear":
        rows = _log(rng, 1, 512)
        k = 8 * _log(rng, 8, 1792)
        n = _log(rng, 64, 28672 if rows <= 16 and k <= 4096 else 8192)
        return dict(kind=kind, rows=rows, n=8 * max(n // 8, 1) if rows > 16 else n, k=k, group=rng.choice([32, 64, 128]), zero=rng.random() < 0.5,
                    bias=rng.random() < 0.3)
    if kind == "attention":
        heads, kv_heads, dim = rng.choice([(14, 2, 64), (16, 8, 128), (24, 8, 128), (32, 8, 128), (12, 12, 64), (8, 1, 128), (8, 4, 256)])
        n = rng.choice([1, 1, 2, 5, _log(rng, 3, 48)])
        lengths = [_log(rng, 1, 32768 // n) for _ in range(n)]
        piece = rng.random() < 0.4   # some bring more than a token
        counts = [min(l, _log(rng, 2, 300)) if piece and i < 2 else 1 for i, l in enumerate(lengths)]
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, lengths=",".join(map(str, lengths)), counts=",".join(map(str, counts)),
                    window=rng.choice([0, 0, _log(rng, 1, 3000)]))
    if kind == "store":
        n = rng.choice([1, 2, _log(rng, 3, 64)])
        return dict(kind=kind, kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128, 256]),
                    firsts=",".join(str(rng.randint(0, 2000)) for _ in range(n)), counts=_sizes(rng, n, 1, max(2048 // n, 2)))
    if kind == "fork":
        return dict(kind=kind, layers=rng.randint(1, 4), kv_heads=rng.choice([1, 2, 4]), dim=rng.choice([64, 128]), n_pages=rng.randint(100, 384),
                    length=_log(rng, 1, 3000), copies=rng.randint(1, 12))
    n = 2 * rng.randint(1, 4)
    return dict(kind=kind, layers=rng.randint(1, 4), kv_heads=rng.choice([1, 2, 4]), dim=rng.choice([64, 128]), n_pages=256,
                lengths=_sizes(rng, n, 1, 12000 // n))


# ------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1))


def _randn(g, *shape, dtype=BF16):
    return torch.randn(*shape, generator=g, device=DEV, dtype=F32).to(dtype)


def _ints(text):
    return [int(v) for v in text.split(",")] if text else []


def _dev(values):
    return torch.tensor(values, device=DEV, dtype=I32)


def _starts(counts):
    s = [0]
    for c in counts:
        s.append(s[-1] + c)
    return _dev(s)


def _linear_inputs(case, seed):
    g = _gen(seed)
    n, k, groups = case["n"], case["k"], -(-case["k"] // case["group"])
    values = (torch.randn(n, k, generator=g, device=DEV, dtype=BF16) * 2.7 + 8).round_().clamp_(0, 15).to(torch.uint8)
    scale = (torch.rand(n, groups, generator=g, device=DEV) * 0.01 + 0.002).to(BF16)
    zero = torch.randint(6, 11, (n, groups), generator=g, device=DEV).to(BF16) if case["zero"] else None
    bias = _randn(g, n) if case["bias"] else None
    return dict(values=values, scale=scale, zero=zero, bias=bias, x=_randn(g, case["rows"], k))


def _rows(g, n, kv_heads, dim):
    """Keys with channels of unequal offset and spread, values around zero."""
    spread = torch.rand(kv_heads, dim, generator=g, device=DEV) * 1.5 + 0.5
    k = torch.randn(n, kv_heads, dim, generator=g, device=DEV) * spread + torch.randn(kv_heads, dim, generator=g, device=DEV)
    return k.to(BF16), _randn(g, n, kv_heads, dim)


def _attention_inputs(case, seed):
    g = _gen(seed)
    lengths, counts = _ints(case["lengths"]), _ints(case["counts"])
    # keys and values of all tokens, sequence behind sequence; the first half of every sequence came in an earlier step
    k, v = _rows(g, sum(max(l, 0) for l in lengths), case["kv_heads"], case["dim"])
    return dict(k=k, v=v, q=_randn(g, sum(counts), case["heads"], case["dim"]), lengths=lengths, counts=counts)


# ------------------------------------------------------------------------------------------------- the operators, plainly
def _linear(x, values, scale, zero, bias, group):
    k = x.shape[1]
    s = scale.float().repeat_interleave(group, 1)[:, :k]
    z = 8.0 if zero is None else zero.float().repeat_interleave(group, 1)[:, :k]
    y = x.float() @ ((values.float() - z) * s).t()
    return (y if bias is None else y + bias.float()).to(BF16)


def _quantise(x):
    """x [..., dim] → values −8 … 7 (int8), scale and middle bf16 [..., dim / 64]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = (hi / 15 - lo / 15).to(BF16)
    middle = (lo + 8 * scale.float()).to(BF16)
    s = scale.float()[..., None]
    values = torch.where(s > 0, ((g - middle.float()[..., None]) / s).round().clamp(-8, 7), torch.zeros_like(g))
    return values.to(torch.int8).flatten(-2), scale, middle


def _read(values, scale, middle):
    return (values.float().unflatten(-1, (-1, GROUP)) * scale.float()[..., None] + middle.float()[..., None]).flatten(-2)


class _Cache:
    """The plain form's cache: a layer's values a byte each, and the bookkeeping as the framework's."""

    def __init__(self, n_pages, n_seqs, max_pages, kv_heads=None, dim=None):
        self.table = torch.full((n_seqs, max_pages), -1, device=DEV, dtype=I32)
        self.length = torch.zeros(n_seqs, device=DEV, dtype=I32)
        self.refs = torch.zeros(n_pages, device=DEV, dtype=I32)
        if kv_heads:
            shape = (n_pages, PAGE, kv_heads, dim)
            small = (n_pages, PAGE, kv_heads, dim // GROUP)
            self.k, self.v = (tuple(torch.zeros(s, device=DEV, dtype=t) for s, t in ((shape, torch.int8), (small, BF16), (small, BF16)))
                              for _ in range(2))

    def extend(self, seqs, counts):
        """Room for counts more tokens of each sequence, in their order while free pages last; the first new position, or −1."""
        seqs = seqs.long()
        length, width = self.length[seqs], self.table.shape[1]
        have, want = (length + PAGE - 1) // PAGE, (length + counts + PAGE - 1) // PAGE
        need = torch.where(want <= width, want - have, torch.zeros_like(want))
        ends = need.cumsum(0)
        free = (self.refs == 0).cumsum(0)
        ok = (want <= width) & ((need == 0) | (ends <= free[-1]))
        column = torch.arange(width, device=DEV)[None]
        new = ok[:, None] & (column >= have[:, None]) & (column < want[:, None])
        number = (ends - need)[:, None] + column - have[:, None]   # which of the free pages
        page = torch.searchsorted(free, (number + 1).clamp(min=1)).to(I32)
        rows = torch.where(new, page, self.table[seqs])
        self.refs.index_add_(0, page.clamp(max=self.refs.shape[0] - 1).long().flatten(), new.to(I32).flatten())
        self.table[seqs] = rows
        self.length[seqs] = length + torch.where(ok, counts, torch.zeros_like(counts))
        return torch.where(ok, length, torch.full_like(length, -1))

    def free(self, seqs):
        rows = self.table[seqs.long()]
        self.refs.index_add_(0, rows.clamp(min=0).long().flatten(), -(rows >= 0).to(I32).flatten())
        self.table[seqs.long()] = -1
        self.length[seqs.long()] = 0

    def fork(self, pages, src, dst):
        """dst (empty) ← src: whole pages are shared, a page that is not full is copied to one of its own; 1, or 0 without a free page."""
        src, dst = src.long(), dst.long()
        length, width = self.length[src], self.table.shape[1]
        whole, part = length // PAGE, (length % PAGE != 0).to(I32)
        ends = part.cumsum(0)
        free = (self.refs == 0).cumsum(0)
        ok = (part == 0) | (ends <= free[-1])
        page = torch.searchsorted(free, ends.clamp(min=1)).to(I32)
        column = torch.arange(width, device=DEV)[None]
        rows = self.table[src]
        shared = ok[:, None] & (column < whole[:, None])
        tail = (ok & (part > 0))[:, None] & (column == whole[:, None])
        source = torch.where(tail, rows, torch.zeros_like(rows)).sum(1)
        rows = torch.where(tail, page[:, None], torch.where(shared, rows, torch.full_like(rows, -1)))
        self.refs.index_add_(0, rows.clamp(min=0).long().flatten(), (rows >= 0).to(I32).flatten())
        self.table[dst] = rows
        self.length[dst] = torch.where(ok, length, torch.zeros_like(length))
        # where there is nothing to copy a page is copied to itself
        target = torch.where(ok & (part > 0), page, torch.zeros_like(page))
        source = torch.where(ok & (part > 0), source.to(I32), torch.zeros_like(page))
        pages[:, target.long()] = pages[:, source.long()]
        return ok.to(I32)

    def compact(self, pages):
        """The pages in use move, in their order, from behind their number into the free ones below it; returns that number."""
        used = self.refs > 0
        n = self.refs.shape[0]
        live = used.sum()
        index = torch.arange(n, device=DEV)
        move, hole = used & (index >= live), ~used & (index < live)
        target = torch.where(move, torch.searchsorted(hole.cumsum(0), move.cumsum(0).clamp(min=1)), index)
        # where every page's content comes from (the last entry takes what does not move)
        source = torch.arange(n + 1, device=DEV).scatter(0, torch.where(move, target, torch.full_like(index, n)), index)[:n]
        pages.copy_(pages[:, source])
        self.refs.copy_(torch.where(move, torch.zeros_like(self.refs), self.refs[source]))
        rows = self.table.clamp(min=0).long()
        self.table.copy_(torch.where(self.table >= 0, target[rows].to(I32), self.table))
        return live.to(I32).reshape(1)

    def place(self, seqs, starts, pos, rows):
        """Page and place in it of every row, and whether the row has one."""
        row = torch.arange(rows, device=DEV, dtype=I32)
        i = (torch.searchsorted(starts, row, right=True) - 1).clamp(max=seqs.shape[0] - 1)
        at = pos[i] + row - starts[i]
        ok = pos[i] >= 0
        at = torch.where(ok, at, torch.zeros_like(at))
        return self.table[seqs[i].long(), (at // PAGE).long()].long(), (at % PAGE).long(), ok

    def store(self, k, v, seqs, starts, pos):
        page, place, _ = self.place(seqs, starts, pos, k.shape[0])
        for held, x in ((self.k, k), (self.v, v)):
            for to, what in zip(held, _quantise(x)):
                to[page, place] = what

    def load(self, seqs, starts, pos, rows):
        page, place, _ = self.place(seqs, starts, pos, rows)
        return tuple(_read(*(h[page, place] for h in held)) for held in (self.k, self.v))

    def attention(self, q, lengths, counts, seqs, pos, window):
        heads, dim = q.shape[1:]
        out, row = torch.zeros_like(q), 0
        for i, (length, count) in enumerate(zip(lengths, counts)):
            if length > 0:
                page = self.table[seqs[i], : -(-length // PAGE)].long()
                k, v = (_read(*(h[page].flatten(0, 1)[:length] for h in held)) for held in (self.k, self.v))
                kv_heads = k.shape[1]
                x = q[row : row + count].float().view(count, kv_heads, -1, dim).permute(1, 2, 0, 3)   # [kv, group, count, dim]
                s = x @ k.permute(1, 2, 0)[:, None] * dim ** -0.5
                at = pos[i] + torch.arange(count, device=DEV)[:, None]
                key = torch.arange(length, device=DEV)[None]
                seen = (key <= at) & (at - key < window) if window else key <= at
                s = s.masked_fill(~seen, float("-inf"))
                s = (s - s.amax(-1, keepdim=True)).exp()
                o = (s @ v.permute(1, 0, 2)[:, None]) / s.sum(-1, keepdim=True)
                out[row : row + count] = o.permute(2, 0, 1, 3).reshape(count, heads, dim).to(BF16)
            row += count
        return out


# ---------------------------------------------------------------------------------------------------------- the interface
def prepare(case, seed):
    if own:
        from tinygpt_b200 import ops
    kind = case["kind"]
    if kind == "linear":
        st = _linear_inputs(case, seed)
        if own:
            st = dict(w=ops.w4_pack(st["values"], st["scale"], st["zero"], group=case["group"]), x=st["x"], bias=st["bias"])
        return dict(case=case, **st)
    if kind == "attention":
        st = _attention_inputs(case, seed)
        n = len(st["lengths"])
        held = [max(l, 0) for l in st["lengths"]]
        half = [l // 2 for l in held]
        n_pages, max_pages = sum(-(-l // PAGE) for l in held) + 3, max(max(-(-l // PAGE) for l in held), 1) + 1
        seqs, rest = _dev(list(range(n))), [a - b for a, b in zip(held, half)]
        if own:
            cache = ops.kv4_cache(1, n_pages, n, max_pages, case["kv_heads"], case["dim"])
            ops.kv4_extend(cache, seqs, _dev(half))
            ops.kv4_extend(cache, seqs, _dev(rest))
            ops.kv4_store(cache, 0, st["k"], st["v"], seqs, _starts(held), torch.zeros_like(seqs))
        else:
            cache = _Cache(n_pages, n, max_pages, case["kv_heads"], case["dim"])
            cache.extend(seqs, _dev(half))
            cache.extend(seqs, _dev(rest))
            cache.store(st["k"], st["v"], seqs, _starts(held), torch.zeros_like(seqs))
        pos = [l - c if l > 0 else -1 for l, c in zip(st["lengths"], st["counts"])]
        return dict(case=case, cache=cache, q=st["q"], seqs=seqs, starts=_starts(st["counts"]), pos=_dev(pos), lengths=st["lengths"],
                    counts=st["counts"], at=pos)
    if kind == "store":
        firsts, counts = _ints(case["firsts"]), _ints(case["counts"])
        g, n = _gen(seed), len(firsts)
        k, v = _rows(g, sum(counts), case["kv_heads"], case["dim"])
        pages = [-(-(f + c) // PAGE) for f, c in zip(firsts, counts)]
        seqs = _dev(list(range(n)))
        cache = (ops.kv4_cache(1, sum(pages) + 1, n, max(pages), case["kv_heads"], case["dim"]) if own else
                 _Cache(sum(pages) + 1, n, max(pages), case["kv_heads"], case["dim"]))
        extend = (lambda c: ops.kv4_extend(cache, seqs, c)) if own else (lambda c: cache.extend(seqs, c))
        extend(_dev(firsts))
        return dict(case=case, cache=cache, k=k, v=v, seqs=seqs, starts=_starts(counts), pos=extend(_dev(counts)))
    g = _gen(seed)
    lengths = [case["length"]] if kind == "fork" else _ints(case["lengths"])
    n = 1 + case["copies"] if kind == "fork" else len(lengths)
    max_pages = max(-(-l // PAGE) for l in lengths) + 1
    page_bytes = 2 * case["kv_heads"] * PAGE * (case["dim"] // 2 + case["dim"] // GROUP * 4)
    pages = torch.randint(0, 256, (case["layers"], case["n_pages"], page_bytes), generator=g, device=DEV, dtype=torch.uint8)
    if own:
        cache = ops.kv4_cache(case["layers"], case["n_pages"], n, max_pages, case["kv_heads"], case["dim"])
        cache.pages.view(pages.shape).copy_(pages)
        extend = lambda s, c: ops.kv4_extend(cache, s, c)
        pages = cache.pages
    else:
        cache = _Cache(case["n_pages"], n, max_pages)
        extend = cache.extend
    if kind == "fork":
        extend(_dev([0]), _dev(lengths))
        dst = _dev(list(range(1, n)))
        return dict(case=case, cache=cache, pages=pages, src=torch.zeros_like(dst), dst=dst, one=torch.ones_like(dst))
    first, second = list(range(0, n, 2)), list(range(1, n, 2))
    halves = [(_dev(h), _dev([lengths[i] for i in h])) for h in (first, second)]
    for s, c in halves:
        extend(s, c)
    return dict(case=case, cache=cache, pages=pages, halves=halves)


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        from tinygpt_b200 import ops
    if kind == "linear":
        if own:
            return ops.linear_w4(state["x"], state["w"], state["bias"])
        return _linear(state["x"], state["values"], state["scale"], state["zero"], state["bias"], case["group"])
    cache = state["cache"]
    if kind == "attention":
        if own:
            return ops.kv4_attention(cache, 0, state["q"], state["seqs"], state["starts"], state["pos"], window=case["window"])
        return cache.attention(state["q"], state["lengths"], state["counts"], state["seqs"], state["at"], case["window"])
    if kind == "store":
        where = state["seqs"], state["starts"], state["pos"]
        if own:
            ops.kv4_store(cache, 0, state["k"], state["v"], *where)
            return ops.kv4_load(cache, 0, *where, state["k"].shape[0])
        cache.store(state["k"], state["v"], *where)
        return cache.load(*where, state["k"].shape[0])
    if kind == "fork":
        if own:
            ops.kv4_free(cache, state["dst"])
            ok = ops.kv4_fork(cache, state["src"], state["dst"])
            pos = ops.kv4_extend(cache, state["dst"], state["one"])
        else:
            cache.free(state["dst"])
            ok = cache.fork(state["pages"], state["src"], state["dst"])
            pos = cache.extend(state["dst"], state["one"])
        return dict(ok=ok, pos=pos, table=cache.table, length=cache.length, refs=cache.refs, pages=state["pages"].view(case["layers"], case["n_pages"], -1))
    out = {}
    for i, (seqs, counts) in enumerate(state["halves"]):
        if own:
            ops.kv4_free(cache, seqs)
            out[f"live{i}"] = ops.kv4_compact(cache)
            out[f"pos{i}"] = ops.kv4_extend(cache, seqs, counts)
        else:
            cache.free(seqs)
            out[f"live{i}"] = cache.compact(state["pages"])
            out[f"pos{i}"] = cache.extend(seqs, counts)
    return dict(out, table=cache.table, length=cache.length, refs=cache.refs, pages=state["pages"].view(case["layers"], case["n_pages"], -1))


def exact(case, seed):
    kind = case["kind"]
    if kind == "linear":
        st = _linear_inputs(case, seed)
        n, k, group = case["n"], case["k"], case["group"]
        y = torch.zeros(case["rows"], n, device=DEV, dtype=F64)
        for j in range(-(-k // group)):   # group by group: scale·(Σ value·x − zero·Σ x)
            cut = slice(j * group, min((j + 1) * group, k))
            x = st["x"][:, cut].double()
            zero = 8.0 if st["zero"] is None else st["zero"][:, j].double()[None]
            y += (x @ st["values"][:, cut].double().t() - x.sum(1, keepdim=True) * zero) * st["scale"][:, j].double()[None]
        return y if st["bias"] is None else y + st["bias"].double()
    if kind == "attention":
        st = _attention_inputs(case, seed)
        k, v = _held(st["k"]), _held(st["v"])
        q, heads, dim = st["q"].double(), case["heads"], case["dim"]
        out = torch.zeros_like(q)
        row = first = 0
        for length, count in zip(st["lengths"], st["counts"]):
            for j in range(count):   # row by row over its own keys
                at = length - count + j
                low = max(0, at - case["window"] + 1) if case["window"] else 0
                if length <= 0:
                    continue
                keys, values = k[first + low : first + at + 1], v[first + low : first + at + 1]
                x = q[row + j].view(case["kv_heads"], heads // case["kv_heads"], dim)
                p = torch.softmax(torch.einsum("hgd,khd->hgk", x, keys) / math.sqrt(dim), -1)
                out[row + j] = torch.einsum("hgk,khd->hgd", p, values).reshape(heads, dim)
            row += count
            first += max(length, 0)
        return out
    if kind == "store":
        k, v = _rows(_gen(seed), sum(_ints(case["counts"])), case["kv_heads"], case["dim"])
        return _held(k), _held(v)
    return None


def _held(x):
    """What the cache holds of x, in 64 bits."""
    g = x.double().view(*x.shape[:-1], -1, GROUP)
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    scale = ((hi - lo) / 15).to(BF16).double()
    middle = (lo + 8 * scale).to(BF16).double()
    steps = torch.where(scale > 0, torch.round((g - middle) / scale.clamp(min=1e-300)), torch.zeros_like(g))
    return (middle + scale * steps.clamp(-8, 7)).view(x.shape)


def work(case):
    kind = case["kind"]
    if kind == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        groups = -(-k // case["group"])
        small = n * groups * (4 if case["zero"] else 2) + (n * 2 if case["bias"] else 0)
        return {"bytes": n * k // 2 + small + rows * (k + n) * 2, "flops": 2 * rows * n * k}
    row_bytes = 0 if kind in ("fork", "compact") else case["kv_heads"] * (case["dim"] // 2 + case["dim"] // GROUP * 4)
    if kind == "attention":
        lengths, counts, window = _ints(case["lengths"]), _ints(case["counts"]), case["window"]
        keys = pairs = 0
        for length, count in zip(lengths, counts):
            if length > 0:
                seen = [min(p + 1, window) if window else p + 1 for p in range(length - count, length)]
                keys += min(length, window + count - 1) if window else length
                pairs += sum(seen)
        return {"bytes": keys * 2 * row_bytes + 2 * sum(counts) * case["heads"] * case["dim"] * 2, "flops": 4 * pairs * case["heads"] * case["dim"]}
    if kind == "store":
        rows = sum(_ints(case["counts"]))
        whole = rows * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * whole * 2 + 2 * 2 * rows * row_bytes + 2 * whole * 4, "flops": 2 * whole * 8}
    page = 2 * case["layers"] * case["kv_heads"] * PAGE * (case["dim"] // 2 + case["dim"] // GROUP * 4)
    if kind == "fork":
        copied = case["copies"] if case["length"] % PAGE else 0
        entries = (case["copies"] + 1) * (-(-case["length"] // PAGE) + 1)
        return {"bytes": 2 * copied * page + 4 * (3 * entries + 2 * case["n_pages"]), "flops": 0}
    lengths = _ints(case["lengths"])
    halves = [sum(-(-l // PAGE) for l in lengths[i::2]) for i in (0, 1)]
    entries = len(lengths) * (max(-(-l // PAGE) for l in lengths) + 1)
    # a half's pages that lie behind the number in use move: the smaller half at most
    return {"bytes": 2 * 2 * min(halves) * page + 4 * (4 * entries + 4 * case["n_pages"]), "flops": 0}
