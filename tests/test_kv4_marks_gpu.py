"""The attention over the paged 4-bit cache counts every token that a row sees once, however the work is cut and its parts are joined (csrc/kv4_attn.cu).

The tokens are marked.  Of the tokens of a span each has +7/8 in one entry that 32 tokens of a step of 32 share, and -1 in another that it shares with one token of
each step; all else is zero.  Such a group is held exactly (scale 1/8, middle 0, values 7, -8 and 0), keys are one whole number a token, held exactly too, and queries
pick it with a scale of ln 2, so that weights are powers of two whose products with a value's scale no rounding to bf16 moves.  Nothing cancels.  So a result is off
by its own rounding (half a step of bf16, 2^-8), by fp32 sums over n tokens (2^-24 each, here and in the sum of the weights) and by what a power of two costs
(2^-16 is ample: scores to 60 times 2^-23) - and a token that is lost or counted twice moves its entries by a 32nd."""
import math

import pytest
import torch

from test_kv4_gpu import dev, starts_of
from tinygpt_b200 import ops

BF16 = torch.bfloat16
STEP = 32


def span(dim):
    return STEP * STEP * (dim // 64)


def keys(length, kv_heads, kind):
    """What a token's keys are, [length]: the power of two of its weight."""
    step = torch.arange(length) // STEP
    power = {"equal": step * 0, "rising": step * 60 // max(length // STEP, 1), "mixed": step * 7 % 11}[kind]
    return power.double()


def values(length, kv_heads, dim, which):
    """Marks of the tokens of span `which`, [length, kv_heads, dim]."""
    v = torch.zeros(length, kv_heads, dim, dtype=torch.float64)
    t = torch.arange(min(which * span(dim), length), min((which + 1) * span(dim), length))
    u = (t - which * span(dim)) // STEP
    for h in range(kv_heads):
        v[t, h, u // 32 * 64 + (u + 5 * h) % 32] = 0.875
        v[t, h, u // 32 * 64 + 32 + (t + 3 * h) % 32] = -1.0
    return v


def expected(power, v, first, rows, heads, window, drop=None, double=None):
    """Rows at positions first ..., their results and bounds; odd heads turn the powers round.  `drop`, `double`: tokens that are lost, or counted twice."""
    n, kv_heads, dim = v.shape
    at, t = first + torch.arange(rows)[:, None], torch.arange(n)[None]
    seen = ((t <= at) & ((at - t < window) | (window == 0))).double()
    if drop is not None:
        seen[:, drop] = 0
    if double is not None:
        seen[:, double] *= 2
    want = torch.zeros(rows, heads, dim, dtype=torch.float64)
    for sign in (0, 1):
        p = seen * 2.0 ** (-power if sign else power)[None]
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
        for h in range(kv_heads):
            mine = [i for i in range(heads) if i // (heads // kv_heads) == h and i % 2 == sign]
            if mine:
                want[:, mine] = (p @ v[:, h])[:, None]
    return want, want.abs() * (2.0 ** -8 + 2.0 ** -16 + 2 * (n + 64) * 2.0 ** -24)


def check(lengths, counts, heads, kv_heads, dim, window=0, room=0, kinds=("equal", "rising", "mixed"), spans=None):
    n = len(lengths)
    cache = ops.kv4_cache(1, sum(-(-l // 64) for l in lengths) + 1, n, max(-(-l // 64) for l in lengths) + room, kv_heads, dim)
    cache.pages.fill_(255)
    seqs, starts = dev(list(range(n))), starts_of(lengths)
    half = [l // 2 for l in lengths]
    ops.kv4_extend(cache, seqs, dev(half))
    ops.kv4_extend(cache, seqs, dev([l - h for l, h in zip(lengths, half)]))
    q = torch.zeros(sum(counts), heads, dim, dtype=BF16, device="cuda")
    q[:, ::2, 0], q[:, 1::2, 0] = 1, -1
    pos = dev([l - c for l, c in zip(lengths, counts)])
    for kind in kinds:
        powers = [keys(l, kv_heads, kind) for l in lengths]
        k = torch.cat(powers).to(BF16).cuda()[:, None, None].expand(-1, kv_heads, dim).contiguous()
        for which in range(-(-max(lengths) // span(dim))) if spans is None else spans:
            v = [values(l, kv_heads, dim, which) for l in lengths]
            ops.kv4_store(cache, 0, k, torch.cat(v).to(BF16).cuda(), seqs, starts, torch.zeros_like(seqs))
            out = ops.kv4_attention(cache, 0, q, seqs, starts_of(counts), pos, scale=math.log(2), window=window).cpu().double()
            row = 0
            for i in range(n):
                want, bound = expected(powers[i], v[i], lengths[i] - counts[i], counts[i], heads, window)
                err = (out[row:row + counts[i]] - want).abs() - bound
                assert bool((err <= 0).all()), (kind, which, i, lengths[i], counts[i], float(err.max()))
                row += counts[i]


@pytest.mark.parametrize("length,rows,dim,window", [(6000, 1, 64, 0), (32768, 1, 128, 0), (2000, 257, 128, 1024), (700, 700, 64, 0)])
def test_no_lost_token_passes(length, rows, dim, window):
    """One token, or a step of them, lost or counted twice, is beyond the bound of the last row, which sees them all (under a window its last ones)."""
    v = values(length, 2, dim, 0)
    for kind in ("equal", "rising", "mixed"):
        power = keys(length, 2, kind)
        want, bound = expected(power, v, length - rows, rows, 2, window)
        top = min(span(dim), length)
        low = max(length - window, 0) if window else 0
        for t in [x for x in (0, 1, 31, 32, 500, low, (low + top) // 2, top - 1) if low <= x < top]:
            for bad in (dict(drop=[t]), dict(double=[t]), dict(drop=list(range(t // 32 * 32, min(t // 32 * 32 + 32, length))))):
                got, _ = expected(power, v, length - rows, rows, 2, window, **bad)
                wrong = (got - want).abs() > bound + got.abs() * 2.0 ** -8
                assert bool(wrong[-1].any(-1).all()), (kind, t, bad)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [([4500], 8, 1, 64), ([9000, 1, 4097], 6, 2, 128), ([8200], 12, 6, 64), ([4200, 4099], 16, 2, 192), ([2500], 2, 1, 256),
                                                        ([900, 33, 64, 1200, 511], 14, 2, 64), ([300 + 7 * i for i in range(18)], 32, 4, 64), ([130, 95, 700] * 20, 2, 2, 128)])
def test_clusters(built_lib, lengths, heads, kv_heads, dim):
    """Sixteen CTAs to one, to a sequence's head."""
    check(lengths, [1] * len(lengths), heads, kv_heads, dim)


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 9000])
@pytest.mark.parametrize("heads,kv_heads,dim", [(6, 2, 64), (24, 8, 128), (3, 1, 192), (4, 2, 256)])
def test_few_rows(built_lib, heads, kv_heads, dim, room):
    """Several blocks of columns to a sequence, one and two tiles of them to a warp; others that bring none."""
    check([1500, 64, 700], [7, 1, 3], heads, kv_heads, dim, room=room, kinds=("mixed",))
    check([333, 1200], [20, 2], heads, kv_heads, dim, window=300, room=room, kinds=("rising",))


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [([6000], 4, 2, 64), ([5000, 64, 2000], 4, 2, 64), ([700] * 40, 4, 2, 64), ([9000], 24, 8, 128), ([7000, 31, 1], 12, 12, 64),
                                                        ([2100, 5000], 6, 2, 192), ([6000], 8, 4, 256), ([64 * i + 1 for i in range(50)], 8, 4, 128)])
def test_even_cut(built_lib, lengths, heads, kv_heads, dim):
    """Pieces that end anywhere in an item, CTAs all inside one, more sequences than a warp has lanes."""
    check(lengths, [1] * len(lengths), heads, kv_heads, dim, room=9000)


@pytest.mark.gpu
def test_a_long_context(built_lib):
    check([32768], [1], 24, 8, 128, kinds=("equal", "rising"), spans=(0, 7, 15))
    check([70001], [1], 4, 1, 64, kinds=("mixed",), spans=(0, 33, 68))


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,counts,heads,kv_heads,dim,window", [([700], [700], 8, 1, 64, 0), ([4353, 1900], [257, 1], 16, 8, 128, 1024), ([520, 900, 1], [520, 333, 1], 6, 2, 128, 0),
                                                                      ([300 + i for i in range(40)], [60] * 40, 8, 2, 64, 90), ([1300], [200], 4, 2, 192, 0), ([1300], [200], 4, 2, 256, 500)])
def test_prompts(built_lib, lengths, counts, heads, kv_heads, dim, window):
    check(lengths, counts, heads, kv_heads, dim, window, kinds=("mixed",))


@pytest.mark.gpu
@pytest.mark.parametrize("piece,room", [(40, 0), (40, 500), (512, 0), (2048, 0)])
def test_a_piece_of_a_prompt_beside_tokens(built_lib, piece, room):
    """A server's step that cuts prompts into pieces: one sequence brings many rows, 63 bring one."""
    check([3000] + [17 + 21 * i for i in range(63)], [piece] + [1] * 63, 16, 4, 64, room=room, kinds=("mixed",), spans=(0, 1))
    check([900] + [3 + 11 * i for i in range(31)], [min(piece, 800)] + [1] * 31, 4, 4, 64, kinds=("rising",))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(40, 1, 64), (71, 1, 128), (128, 2, 64), (150, 1, 64)])
def test_many_query_heads_to_a_key_value_head(built_lib, heads, kv_heads, dim):
    """More columns of a single token than two tiles: the prompts' way."""
    check([1, 777, 2000, 64], [1, 1, 1, 1], heads, kv_heads, dim, kinds=("equal", "mixed"))
    check([600, 90], [2, 1], heads, kv_heads, dim, window=100, kinds=("rising",))
