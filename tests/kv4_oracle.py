"""The paged cache of 4-bit keys and values, plainly: quantisation (in the fp32 steps of its definition), attention in 64 bits with the bound of the kernel's
error, and the bookkeeping of pages as lists."""
import torch

BF16 = torch.bfloat16
PAGE, GROUP = 64, 64


def held(x):
    """What a cache holds of x [..., dim] bf16, fp32 (CPU)."""
    g = x.cpu().float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = (hi / 15 - lo / 15).to(BF16).float()
    m = (lo + 8 * s).to(BF16).float()
    n = torch.where(s > 0, ((g - m) / torch.where(s > 0, s, torch.ones_like(s))).round().clamp(-8, 7), torch.zeros_like(g))
    out = m + s * n
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    return torch.where(bad, torch.full_like(out, float("nan")), out).flatten(-2)


def attention(q, k, v, first, scale, window):
    """q [rows, heads, dim] at positions first …, over k, v [keys, kv_heads, dim] (fp32): the result in 64 bits and the bound of the error.
    The bound: a weight times its value's scale is rounded to bf16 (half a step, 2^-8 of it; scale·value is at most the group's range), the
    result is rounded to bf16, and a score's fp32 sums (dim + 8 roundings of its terms' magnitudes) enter the weights' ratio twice."""
    rows, heads, dim = q.shape
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    out, bound = torch.zeros(rows, heads, dim, dtype=torch.float64), torch.zeros(rows, heads, dim, dtype=torch.float64)
    group = heads // k.shape[1]
    spread = v.unflatten(-1, (-1, GROUP))
    spread = (spread.amax(-1, keepdim=True) - spread.amin(-1, keepdim=True)).expand_as(spread).flatten(-2)
    for j in range(rows):
        at = first + j
        low, high = max(0, at - window + 1) if window else 0, min(at + 1, k.shape[0])
        if at < 0 or low >= high:
            continue
        for h in range(heads):
            keys, vals = k[low:high, h // group], v[low:high, h // group]
            s = keys @ q[j, h] * scale
            size = float((keys.abs() @ q[j, h].abs()).max()) * scale
            p = torch.softmax(s, 0)
            out[j, h] = p @ vals
            delta = size * (dim + 8) * 2.0 ** -23 + 2.0 ** -19
            bound[j, h] = 2.0 ** -8 * (out[j, h].abs() + p @ spread[low:high, h // group]) + 4 * delta * (p @ vals.abs())
    return out, bound


class Pages:
    """The bookkeeping, a sequence as a list of pages."""

    def __init__(self, n_pages, n_seqs, max_pages):
        self.seqs = [[] for _ in range(n_seqs)]
        self.length = [0] * n_seqs
        self.refs = [0] * n_pages
        self.max_pages = max_pages
        self.copied = []   # (from, to) since last asked

    def _free(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def extend(self, seqs, counts):
        free, used, out, seen = self._free(), 0, [], set()
        for s, c in zip(seqs, counts):
            if not 0 <= s < len(self.seqs) or s in seen or c < 0:
                out.append(-1)
                seen.add(s)
                continue
            seen.add(s)
            want = -(-(self.length[s] + c) // PAGE)
            if want > self.max_pages:
                out.append(-1)
                continue
            need = want - len(self.seqs[s])
            used += need
            if need and used > len(free):
                out.append(-1)
                continue
            for p in free[used - need:used]:
                self.seqs[s].append(p)
                self.refs[p] = 1
            out.append(self.length[s])
            self.length[s] += c
        return out

    def fork(self, src, dst):
        free, used, out, seen = self._free(), 0, [], set()
        was = [(list(p), l) for p, l in zip(self.seqs, self.length)]
        n = len(was)
        for s, d in zip(src, dst):
            ok = 0 <= s < n and 0 <= d < n and s != d and d not in seen and was[d][1] == 0
            seen.add(d)
            if not ok:
                out.append(0)
                continue
            pages, length = was[s]
            part = length % PAGE != 0
            used += part
            if part and used > len(free):
                out.append(0)
                continue
            mine = pages[:length // PAGE]
            for p in mine:
                self.refs[p] += 1
            if part:
                self.copied.append((pages[length // PAGE], free[used - 1]))
                mine = mine + [free[used - 1]]
                self.refs[free[used - 1]] = 1
            self.seqs[d], self.length[d] = mine, length
            out.append(1)
        return out

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.seqs):
                for p in self.seqs[s]:
                    self.refs[p] -= 1
                self.seqs[s], self.length[s] = [], 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        moves = dict(zip([p for p in range(live, len(self.refs)) if self.refs[p]], holes))
        for a, b in moves.items():
            self.refs[a], self.refs[b] = 0, self.refs[a]
            self.copied.append((a, b))
        self.seqs = [[moves.get(p, p) for p in s] for s in self.seqs]
        return live

    def check(self, cache):
        table = [s + [-1] * (self.max_pages - len(s)) for s in self.seqs]
        assert cache.table.tolist() == table and cache.length.tolist() == self.length and cache.refs.tolist() == self.refs
