"""The operators of serving in 8 bits and of experts, as measurable cases: norms whose result leaves in 8-bit floating point with a scale for every 128
entries, Linears over weights of 8 bits with a scale for every block of 128 × 128, products of rows grouped by expert (bf16 and 8 bits), and a layer of
routed experts as a whole.

Rows in 8 bits (e4m3): of a block of 128 entries t, s = max(fp32(max|t| / 448), 2^-126), value = e4m3(fp32(t / s)), and what is read is value·scale.  The
scale is s; a norm's is s·rsqrt(mean(z²) + eps) with t = z·weight, z the row or its bf16 sum with the residual (which is handed out too).
Weights in 8 bits: W[i, j] = scale[i // 128, j // 128]·value[i, j].
Groups: rows starts[e] … starts[e + 1] − 1 meet the matrix of expert e; rows behind the last group come out as zeros.
Experts: a row's chosen experts each make W_out·(silu(g)·u) of [g | u] = W_in·row, the row, the product of [g | u] (a bf16) and silu(g)·u as 8-bit rows; the
bf16 results are summed with the row's weights in the order in which they were chosen.
A case is a dict of plain values whose "kind" says which operator it calls.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16, F32, F64, I32, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.float8_e4m3fn
BLOCK, TOP = 128, 448.0
EPS = 1e-6


def listed():
    return [
        # the smallest call: the norm between two blocks of a small model while it decodes one token
        dict(name="norm_token", kind="norm", rows=1, dim=896, residual=True),
        # the same norm over a long prompt of a large model
        dict(name="norm_prompt", kind="norm", rows=4096, dim=4096, residual=True),
        # a first layer's norm (no residual yet) of a ragged batch, a width that ends inside a block
        dict(name="norm_odd", kind="norm", rows=333, dim=1000, residual=False),
        # one decoded row through the merged q | k | v of a small model, with its bias, from bf16
        dict(name="linear_small", kind="linear", rows=1, n=1152, k=896, bias=True, given=False),
        # one decoded row through the merged gate | up of a large model, behind a norm that handed out 8 bits: the weight stream itself
        dict(name="linear_token", kind="linear", rows=1, n=28672, k=4096, bias=False, given=True),
        # a decode batch through a down-projection, from bf16
        dict(name="linear_batch", kind="linear", rows=48, n=4096, k=14336, bias=False, given=False),
        # a long prompt through the merged gate | up
        dict(name="linear_prompt", kind="linear", rows=4096, n=28672, k=4096, bias=False, given=True),
        # one token's four chosen experts of 32, bf16 weights: the streams of four matrices
        dict(name="group_token", kind="group", eight=False, n=2048, k=2048, behind=0, counts=",".join("1" if e in (3, 4, 17, 30) else "0" for e in range(32))),
        # a prompt's rows over 32 experts as a router shares them out, bf16 weights
        dict(name="group_prompt", kind="group", eight=False, n=2048, k=2048, behind=0, counts=_shares(8192, 32)),
        # a middling batch in 8 bits: experts without a row, with one, with many; sizes that end inside a block; rows behind the last group
        dict(name="group_ragged", kind="group", eight=True, n=1100, k=2056, behind=7, counts="0,1,300,17,0,64,129,5,0,0,33,2,256,90,1,0"),
        # a decode step of eight sequences through a layer of 32 experts, four a token
        dict(name="experts_batch", kind="experts", rows=8, top=4, experts=32, width=2048, ff=1024),
        # a prompt through the same layer
        dict(name="experts_prompt", kind="experts", rows=2048, top=4, experts=32, width=2048, ff=1024),
    ]


def _shares(rows, experts):
    """Rows of each expert where a router prefers some: shares falling by a fourth from the first to the eighth of every eight."""
    part = [1.25 ** -(e * 5 % 8) for e in range(experts)]
    counts = [int(rows * p / sum(part)) for p in part]
    counts[0] += rows - sum(counts)
    return ",".join(map(str, counts))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "linear", "linear", "group", "group", "experts"])
    if kind == "norm":
        return dict(kind=kind, rows=_log(rng, 1, 4096), dim=_log(rng, 64, 8192), residual=rng.random() < 0.7)
    if kind == "linear":
        rows, k = _log(rng, 1, 4096), _log(rng, 64, 14336)
        return dict(kind=kind, rows=rows, n=_log(rng, 64, 28672 if k <= 4096 else 8192), k=k, bias=rng.random() < 0.3, given=rng.random() < 0.5)
    if kind == "group":
        experts = _log(rng, 2, 64)
        rows = _log(rng, 1, 8192)
        favour = [rng.random() ** 2 * (rng.random() < 0.8) + 1e-6 for _ in range(experts)]
        counts = [0] * experts
        for e in rng.choices(range(experts), favour, k=rows):
            counts[e] += 1
        eight = rng.random() < 0.5
        k = _log(rng, 64, 2048)
        return dict(kind=kind, eight=eight, n=_log(rng, 64, 2048), k=k if eight else 8 * (k // 8), behind=rng.choice([0, 0, 5, 40]),
                    counts=",".join(map(str, counts)))
    experts = _log(rng, 4, 64)
    return dict(kind=kind, rows=_log(rng, 1, 2048), top=rng.randint(1, min(8, experts)), experts=experts, width=_log(rng, 128, 2048), ff=_log(rng, 64, 1024))


# ------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1))


def _randn(g, *shape, dtype=BF16):
    return torch.randn(*shape, generator=g, device=DEV, dtype=F32).to(dtype)


def _rows(g, rows, dim):
    """Activations: channels of unequal spread, some of them large."""
    spread = torch.exp(torch.randn(dim, generator=g, device=DEV) * 0.5)
    return (torch.randn(rows, dim, generator=g, device=DEV) * spread).to(BF16)


def _weight(g, *shape):
    """Values and scales as a checkpoint in 8 bits holds them: a block's largest value is near 448, scales differ from block to block."""
    *lead, n, k = shape
    values = (torch.randn(*shape, generator=g, device=DEV, dtype=BF16) * 110).clamp_(-TOP, TOP).to(E4M3)
    scale = torch.exp(torch.randn(*lead, -(-n // BLOCK), -(-k // BLOCK), generator=g, device=DEV) * 0.2) / (110 * math.sqrt(k))
    return values, scale


def _ints(text):
    return [int(v) for v in text.split(",")]


def _inputs(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "norm":
        shape = case["rows"], case["dim"]
        weight = (1 + 0.2 * torch.randn(case["dim"], generator=g, device=DEV)).to(BF16)
        return dict(x=_randn(g, *shape), residual=_rows(g, *shape) if case["residual"] else None, weight=weight)
    if kind == "linear":
        values, scale = _weight(g, case["n"], case["k"])
        return dict(x=_rows(g, case["rows"], case["k"]), values=values, scale=scale, bias=_randn(g, case["n"]) if case["bias"] else None)
    if kind == "group":
        counts = _ints(case["counts"])
        starts = torch.tensor([0] + counts, device=DEV).cumsum(0).to(I32)
        st = dict(x=_rows(g, sum(counts) + case["behind"], case["k"]), starts=starts, counts=counts)
        shape = len(counts), case["n"], case["k"]
        if case["eight"]:
            st["values"], st["scale"] = _weight(g, *shape)
        else:
            st["weight"] = torch.randn(*shape, generator=g, device=DEV, dtype=BF16) / math.sqrt(case["k"])
        return st
    rows, experts, width, ff = case["rows"], case["experts"], case["width"], case["ff"]
    logits = torch.randn(rows, experts, generator=g, device=DEV) + 0.7 * torch.randn(experts, generator=g, device=DEV)
    best = logits.topk(case["top"], dim=1)
    return dict(x=_rows(g, rows, width), chosen=best.indices.to(I32), weights=torch.softmax(best.values, 1), w_in=_weight(g, experts, 2 * ff, width),
                w_out=_weight(g, experts, width, ff))


# ------------------------------------------------------------------------------------------------- the operators, plainly
def _blocks(t):
    """[rows, k] → [rows, blocks, 128], zeros behind the end."""
    return torch.nn.functional.pad(t, (0, -t.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK))


def _eight(t):
    """fp32 rows → (values as fp32 [rows, k], s [rows, blocks])."""
    b = _blocks(t)
    # (a quotient by a plain number may be a product with its reciprocal, which is another number now and then)
    s = (b.abs().amax(-1) / torch.full_like(b[..., 0], TOP)).clamp(min=2.0 ** -126)
    return (b / s[..., None]).clamp(-TOP, TOP).to(E4M3).float().flatten(1)[:, : t.shape[1]], s


def _spread(scale, k):
    """A number for every block → one for every column."""
    return scale.repeat_interleave(BLOCK, -1)[..., :k]


def _wide(values, scale):
    n, k = values.shape[-2:]
    return values.float() * _spread(scale.repeat_interleave(BLOCK, -2)[..., :n, :], k)


def _read(values, s):
    return values * _spread(s, values.shape[1])


def _grouped(x, matrix, counts, n):
    y = torch.zeros(x.shape[0], n, device=DEV, dtype=BF16)
    row = 0
    for e, count in enumerate(counts):
        if count:
            y[row : row + count] = (x[row : row + count] @ matrix(e).t()).to(BF16)
            row += count
    return y


def _plain(st, case):
    kind = case["kind"]
    if kind == "norm":
        x, residual = st["x"], st["residual"]
        z = x.float() if residual is None else (x.float() + residual.float()).to(BF16).float()
        inv = torch.rsqrt(z.square().mean(1, keepdim=True) + EPS)
        values, s = _eight(z * st["weight"].float())
        out = _read(values, s * inv)
        return out if residual is None else (out, z.to(BF16))
    if kind == "linear":
        x = _read(*st["rows"]) if case["given"] else _read(*_eight(st["x"].float()))
        y = x @ _wide(st["values"], st["scale"]).t()
        return (y if st["bias"] is None else y + st["bias"].float()).to(BF16)
    if kind == "group":
        if case["eight"]:
            return _grouped(_read(*_eight(st["x"].float())), lambda e: _wide(st["values"][e], st["scale"][e]), st["counts"], case["n"])
        return _grouped(st["x"].float(), lambda e: st["weight"][e].float(), st["counts"], case["n"])
    rows, top, ff = case["rows"], case["top"], case["ff"]
    order = torch.argsort(st["chosen"].flatten(), stable=True)
    x = _read(*_eight(st["x"].float()))[order // top]
    (v_in, s_in), (v_out, s_out) = st["w_in"], st["w_out"]
    gu = _grouped(x, lambda e: _wide(v_in[e], s_in[e]), st["counts"], 2 * ff).float()
    g, u = gu[:, :ff], gu[:, ff:]
    a = _read(*_eight(g / (1 + torch.exp(-g)) * u))
    y = _grouped(a, lambda e: _wide(v_out[e], s_out[e]), st["counts"], case["width"]).float()
    back = torch.empty_like(y)
    back[order] = y
    return (back.unflatten(0, (rows, top)) * st["weights"][..., None]).sum(1).to(BF16)


# ---------------------------------------------------------------------------------------------------------- the interface
def prepare(case, seed):
    st, kind = _inputs(case, seed), case["kind"]
    if own:
        from tinygpt_b200 import ops
        if kind == "linear":
            st["w"] = ops.f8_pack(st.pop("values"), st.pop("scale"))
            if case["given"]:
                st["x"] = ops.f8_rows(st["x"])
        elif kind == "group" and case["eight"]:
            st["w"] = ops.f8_pack(st.pop("values"), st.pop("scale"))
        elif kind == "experts":
            st["w_in"], st["w_out"] = ops.f8_pack(*st["w_in"]), ops.f8_pack(*st["w_out"])
    elif kind == "linear" and case["given"]:
        st["rows"] = _eight(st["x"].float())
    elif kind == "experts":
        st["counts"] = torch.bincount(st["chosen"].flatten(), minlength=case["experts"]).tolist()
    return dict(case=case, **st)


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        return _plain(state, case)
    from tinygpt_b200 import ops
    if kind == "norm":
        if state["residual"] is None:
            return ops.f8_rows_dequantize(ops.rms_norm_f8(state["x"], state["weight"], EPS))
        rows, z = ops.add_rms_norm_f8(state["x"], state["residual"], state["weight"], EPS)
        return ops.f8_rows_dequantize(rows), z
    if kind == "linear":
        return ops.linear_f8(state["x"], state["w"], state["bias"])
    if kind == "group":
        if case["eight"]:
            return ops.grouped_linear_f8(state["x"], state["w"], state["starts"])
        return ops.grouped_linear(state["x"], state["weight"], state["starts"])
    return ops.experts_f8(state["x"], state["chosen"], state["weights"], state["w_in"], state["w_out"])


# ------------------------------------------------------------------------------------------------------ in 64 bits, apart
def _e4m3(v):
    """The nearest number of the format, ties to even: steps of 2^-9 up to 2^-6, then of an eighth of the power of two."""
    step = torch.exp2((torch.frexp(v).exponent - 1).clamp(min=-6).double() - 3)
    return ((v / step).round() * step).clamp(-TOP, TOP)


def _held(t, factor=None):
    """What 8-bit rows hold of t, in 64 bits; a scale is an fp32 number, and so is the quotient that is rounded: three quarters of a block's largest
    entry, a common ratio, lie half-way between two numbers of the format."""
    out = torch.empty_like(t, dtype=F64)
    for j in range(0, t.shape[1], BLOCK):
        b = t[:, j : j + BLOCK].double()
        largest = b.abs().max(1, keepdim=True).values
        s = (largest / torch.full_like(largest, TOP)).float().double().clamp(min=2.0 ** -126)
        out[:, j : j + BLOCK] = _e4m3((b / s).float().double()) * (s if factor is None else s * factor)
    return out


def _matrix(values, scale):
    w = values.double()
    for i in range(scale.shape[0]):
        for j in range(scale.shape[1]):
            w[i * BLOCK : (i + 1) * BLOCK, j * BLOCK : (j + 1) * BLOCK] *= scale[i, j].double()
    return w


def exact(case, seed):
    st, kind = _inputs(case, seed), case["kind"]
    if kind == "norm":
        z = st["x"].double()
        if st["residual"] is not None:
            z = (z + st["residual"].double()).to(BF16).double()
        out = _held(z * st["weight"].double(), 1 / torch.sqrt((z * z).mean(1, keepdim=True) + EPS))
        return out if st["residual"] is None else (out, z)
    if kind == "linear":
        y = _held(st["x"]) @ _matrix(st["values"], st["scale"]).t()
        return y if st["bias"] is None else y + st["bias"].double()
    if kind == "group":
        x = _held(st["x"]) if case["eight"] else st["x"].double()
        y = torch.zeros(x.shape[0], case["n"], device=DEV, dtype=F64)
        starts = st["starts"].tolist()
        for e in range(len(starts) - 1):
            a, b = starts[e], starts[e + 1]
            if a < b:
                y[a:b] = x[a:b] @ (_matrix(st["values"][e], st["scale"][e]) if case["eight"] else st["weight"][e].double()).t()
        return y
    x, ff = _held(st["x"]), case["ff"]
    y = torch.zeros(case["rows"], case["width"], device=DEV, dtype=F64)
    for e in range(case["experts"]):
        row, t = (st["chosen"] == e).nonzero(as_tuple=True)
        if len(row):
            gu = (x[row] @ _matrix(st["w_in"][0][e], st["w_in"][1][e]).t()).to(BF16).double()
            a = _held(torch.nn.functional.silu(gu[:, :ff]) * gu[:, ff:])
            part = (a @ _matrix(st["w_out"][0][e], st["w_out"][1][e]).t()).to(BF16).double()
            y.index_add_(0, row, part * st["weights"][row, t].double()[:, None])
    return y


def work(case):
    kind = case["kind"]
    eight = lambda rows, dim: rows * dim + 4 * rows * -(-dim // BLOCK)
    matrix = lambda n, k: n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK)
    if kind == "norm":
        rows, dim = case["rows"], case["dim"]
        # in: the row, its residual and the weight; out: the sum, 8 bits and scales — which are read again and written as fp32
        return {"bytes": rows * dim * 2 * (3 if case["residual"] else 1) + 2 * dim + 2 * eight(rows, dim) + 4 * rows * dim, "flops": 8 * rows * dim}
    if kind == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": matrix(n, k) + (eight(rows, k) if case["given"] else 2 * rows * k) + 2 * rows * n + (2 * n if case["bias"] else 0),
                "flops": 2 * rows * n * k}
    if kind == "group":
        counts, n, k = _ints(case["counts"]), case["n"], case["k"]
        rows, used = sum(counts), sum(c > 0 for c in counts)
        return {"bytes": used * (matrix(n, k) if case["eight"] else 2 * n * k) + 2 * rows * k + 2 * (rows + case["behind"]) * n, "flops": 2 * rows * n * k}
    rows, top, experts, width, ff = (case[name] for name in ("rows", "top", "experts", "width", "ff"))
    used = max(min(top, experts), int(experts * (1 - (1 - top / experts) ** rows)))   # experts that some row chose, as rows choose apart from each other
    return {"bytes": used * (matrix(2 * ff, width) + matrix(width, ff)) + rows * width * 4 + rows * top * 8, "flops": 6 * rows * top * width * ff}
