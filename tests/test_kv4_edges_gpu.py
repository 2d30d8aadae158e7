"""The paged cache of 4-bit keys and values where it can go wrong: windows behind all of a sequence whose row of the table is full."""
import pytest
import torch

import kv4_oracle as orc
from test_kv4_gpu import Rand, dev, filled, starts_of
from tinygpt_b200 import ops

BF16 = torch.bfloat16


# ------------------------------------------------------------------------------------------------- full rows of the table
@pytest.mark.gpu
@pytest.mark.parametrize("pages,rows", [(1, 1), (3, 1), (300, 1), (300, 6), (3, 50), (40, 50)])   # clusters, the even cut, blocks for a CTA
def test_windows_behind_a_full_row(built_lib, pages, rows):
    """The last sequence fills its row of the table, which lies in front of other numbers; rows that see its last tokens or nothing."""
    rand, heads, dim, length = Rand(21), 4, 64, 64 * pages
    plain = ops.kv4_cache(1, 2 * pages + 4, 2, pages, 1, dim)
    numbers = torch.full((2 * pages + 8,), 2 * pages + 3, dtype=torch.int32, device="cuda")   # a page of NaN, behind the table
    numbers[:2 * pages] = torch.arange(2 * pages, device="cuda", dtype=torch.int32).flip(0)
    cache = ops.KV4Cache(plain.pages, numbers[:2 * pages].view(2, pages), plain.length, plain.refs, 1, dim)
    cache.pages.fill_(255)
    cache.refs[:2 * pages] = 1
    cache.length.copy_(dev([length, length]))
    k, v = rand(2 * length, 1, dim), rand(2 * length, 1, dim)
    ops.kv4_store(cache, 0, k, v, dev([0, 1]), dev([0, length, 2 * length]), dev([0, 0]))
    hk, hv, q = orc.held(k), orc.held(v), rand(2 * rows, heads, dim)
    for window in (1, 33, 64):
        for at in (length - rows, length, length + window - 1 - rows // 2, length + window - 2, length + window - 1, length + window, length + 5000):
            out = ops.kv4_attention(cache, 0, q, dev([0, 1]), dev([0, rows, 2 * rows]), dev([at, at]), window=window).cpu().double()
            for s in (0, 1):
                mine = slice(s * length, (s + 1) * length)
                want, bound = orc.attention(q[s * rows:(s + 1) * rows], hk[mine], hv[mine], at, dim ** -0.5, window)
                got = out[s * rows:(s + 1) * rows]
                assert bool(((got - want).abs() <= bound).all()), (window, at, s)
                blind = max(0, min(rows, at + rows - (length + window - 1)))
                assert blind == 0 or not got[rows - blind:].any()
