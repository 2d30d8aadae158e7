"""Rows and weights of 8 bits and routed experts in 64 bits, from their definitions."""
import torch

F8 = torch.float8_e4m3fn


def e4m3(v):
    """The nearest number of the format to fp64 numbers, ties to even, at most ±448: steps of 2^-9 up to 2^-6, then of an eighth of the power of two."""
    step = torch.exp2((torch.frexp(v).exponent - 1).clamp(min=-6).double() - 3)
    return ((v / step).round() * step).clamp(-448, 448)


def cut(t):
    """[rows, k] → [rows, blocks, 128]"""
    return torch.nn.functional.pad(t, (0, -t.shape[1] % 128)).unflatten(1, (-1, 128))


def scales(t):
    """fp32 scale of every block, [rows, blocks]; t fp64 (numbers that fp32 holds)"""
    return (cut(t).abs().amax(-1) / 448).float().clamp(min=2.0 ** -126)


def eight(t):
    """t fp64 [rows, k] → (values fp64 [rows, k], scales fp32 [rows, blocks])"""
    s = scales(t)
    return e4m3((cut(t) / s.double()[..., None]).float().double()).flatten(1)[:, : t.shape[1]], s


def spread(s, k):
    return s.double().repeat_interleave(128, 1)[:, :k]


def held(rows):
    """What F8Rows stand for, fp64 [rows, k]"""
    q = rows.q.reshape(-1, rows.q.shape[-1])[:, : rows.k].double()
    return q * spread(rows.scale.t(), rows.k)


def dense(w):
    """What an F8Weight stands for, fp64"""
    s = w.scale.double().repeat_interleave(128, -2)[..., : w.n, :].repeat_interleave(128, -1)[..., : w.k]
    return w.q[..., : w.k].double() * s


def close(got, x, w, bias=None):
    """|error| ≤ half a step of bf16 of the result + the fp32 sums': every product exact, no more than a rounding for each term and each block's factor and
    sum, of the terms' sum of magnitudes; 32 terms more for what a tensor core drops when it lines a product's terms up."""
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    bound = want.abs() * 2.0 ** -8 + size * ((x.shape[1] + 32) * 2.0 ** -23) + 1e-38
    worst = ((got.double() - want).abs() / bound).max() if got.numel() else torch.zeros(())
    assert bool(((got.double() - want).abs() <= bound).all()), float(worst)
    return float(worst)


def order(chosen, experts):
    """starts, source, place of a stable sort, as lists"""
    rows, top = chosen.shape
    flat = chosen.flatten().tolist()
    pairs = [i for e in range(experts) for i, c in enumerate(flat) if c == e]
    starts = [0]
    for e in range(experts):
        starts.append(starts[-1] + sum(c == e for c in flat))
    place = [-1] * len(flat)
    for at, i in enumerate(pairs):
        place[i] = at
    return starts, [i // top for i in pairs] + [-1] * (len(flat) - len(pairs)), place
