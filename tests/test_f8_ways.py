"""Every way that a product of csrc/group_gemm.cu can be cut — tiles of 16 to 128 rows beside 128 channels and the wide ones, one to eight CTAs to a tile — by itself: the
library says which way a call of given sizes takes (b200_product_way), and the smallest call of each way meets the definition in 64 bits."""
import ctypes as C
import functools

import pytest
import torch

import f8_oracle as orc
from test_f8_gpu import BF16, I32, each_group, gen, randn, weight
from tinygpt_b200 import ops

WAYS = [(rows, ctas) for rows in (16, 32, 64, 128) for ctas in (1, 2, 4, 8)] + [(0, 1)]
KINDS = ("linear_f8", "grouped_f8", "grouped_bf16")
ROWS = (1, 3, 5, 9, 17, 24, 33, 47, 50, 65, 80, 99, 130, 160, 200, 260, 300, 400, 523, 700, 1000, 1500, 2003, 3000)
EVEN = (72, 136, 264, 520, 1000, 2000, 4096), (264, 520, 1032, 2064, 4104, 8208, 14352)   # channels, k: rows of y that take 16-byte stores
ODD = (75, 131, 261, 515, 1003, 2049, 4099), (131, 393, 1001, 2103, 4001, 8009, 14001)    # and that take none, k off the blocks of 128 and of 16


def way(rows, experts, n, k, eight):
    from tinygpt_b200._lib import check, lib
    tile, ctas = C.c_int32(-1), C.c_int32(-1)
    check(lib().b200_product_way(rows, experts, n, k, eight, C.byref(tile), C.byref(ctas)), "b200_product_way")
    return tile.value, ctas.value


@functools.lru_cache(None)
def smallest(kind, odd):
    """way → (rows, experts, n, k) of the cheapest call among the sizes above that takes it"""
    eight, best = kind != "grouped_bf16", {}
    ns, ks = ODD if odd else EVEN
    for rows in ROWS:
        for experts in (0,) if kind == "linear_f8" else (2, 3, 5, 8, 16, 32):
            for n in ns:
                for k in ks:
                    k -= 0 if eight else k % 8
                    cost = max(experts, 1) * n * k + 30 * rows * n + rows * k
                    w = way(rows, experts, n, k, eight)
                    if w not in best or cost < best[w][0]:
                        best[w] = cost, (rows, experts, n, k)
    return {w: sizes for w, (_, sizes) in best.items()}


def test_which_ways_there_are(built_lib):
    for kind in KINDS:
        found = set(smallest(kind, False)) | set(smallest(kind, True))
        assert found <= set(WAYS) and {rows for rows, _ in found} == {0, 16, 32, 64, 128} and {ctas for _, ctas in found} == {1, 2, 4, 8}
    from tinygpt_b200._lib import lib
    a, b = C.c_int32(-1), C.c_int32(-1)
    for bad in ((0, 4, 8, 8, 1), (1 << 24, 4, 8, 8, 1), (1, 1025, 8, 8, 1), (1, -1, 8, 8, 1), (1, 4, 0, 8, 1), (1, 4, 1 << 21, 8, 1), (1, 4, 8, 0, 1), (1, 4, 8, (1 << 24) + 1, 1),
                (1, 1024, 1 << 21, 8, 1), (1, 0, 8, 8, 0)):
        assert lib().b200_product_way(*bad, C.byref(a), C.byref(b)) != 0 and (a.value, b.value) == (-1, -1), bad
    assert lib().b200_product_way(1, 4, 8, 8, 1, None, C.byref(b)) != 0 and lib().b200_product_way(1, 4, 8, 8, 1, C.byref(a), None) != 0


def cut_rows(rows, experts, seed):
    """starts of uneven groups — none, one and many rows — with a row in front of the first and two behind the last where there are enough"""
    before, behind = (1, 2) if rows > 8 else (0, 0)
    share = torch.rand(experts, generator=torch.Generator().manual_seed(seed)) ** 2
    if experts > 2 and rows > 8:
        share[1] = 0
    of = torch.multinomial(share, rows - before - behind, replacement=True, generator=torch.Generator().manual_seed(seed))
    counts = torch.bincount(of, minlength=experts)
    return torch.cat([torch.tensor([before]), before + counts.cumsum(0)]).to(I32).cuda()


def call_of(kind, which, odd):
    sizes = smallest(kind, odd).get(which)
    if sizes is None:
        pytest.skip("no call of these sizes is cut so")
    assert way(*sizes, kind != "grouped_bf16") == which
    return sizes


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [False, True], ids=["even", "odd"])
@pytest.mark.parametrize("which", WAYS, ids=lambda w: f"{w[0] or 'wide'}x{w[1]}")
@pytest.mark.parametrize("kind", KINDS)
def test_against_64_bits(built_lib, kind, which, odd):
    rows, experts, n, k = call_of(kind, which, odd)
    x, bias = randn(rows, k, seed=rows), randn(n, seed=5)
    if kind == "linear_f8":
        w, x8 = weight(n, k, seed=n), ops.f8_rows(x)
        held, full = orc.held(x8), orc.dense(w)
        y = ops.linear_f8(x8, w)
        orc.close(y, held, full)
        orc.close(ops.linear_f8(x8, w, bias), held, full, bias)
        assert torch.equal(ops.linear_f8(x, w), y)   # from bf16 rows, W read ahead
        return
    starts = cut_rows(rows, experts, seed=n)
    if kind == "grouped_f8":
        w, x8 = weight(n, k, experts, seed=n), ops.f8_rows(x)
        y = ops.grouped_linear_f8(x8, w, starts)
        each_group(y, orc.held(x8), orc.dense(w), starts)
        assert torch.equal(ops.grouped_linear_f8(x, w, starts), y)
    else:
        w = (torch.randn(experts, n, k, generator=gen(n), device="cuda") / k ** 0.5).to(BF16)
        each_group(ops.grouped_linear(x, w, starts), x.double(), w.double(), starts)


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [False, True], ids=["even", "odd"])
@pytest.mark.parametrize("which", WAYS, ids=lambda w: f"{w[0] or 'wide'}x{w[1]}")
@pytest.mark.parametrize("kind", KINDS)
def test_sums_that_are_exact(built_lib, kind, which, odd):
    """Whole numbers whose sums fp32 holds (below 2^24): every term counts once, in any order, and one rounding to bf16 is left."""
    rows, experts, n, k = call_of(kind, which, odd)
    g = gen(rows + n)
    x = torch.zeros(rows, k, device="cuda", dtype=BF16)
    x[:, ::7] = torch.randint(-1, 2, (rows, len(range(0, k, 7))), generator=g, device="cuda").to(BF16)
    x[:, 0::128] = 448   # the block's scale is 1
    v = torch.randint(-1, 2, (max(experts, 1), n, k), generator=g, device="cuda").to(torch.int8)
    if kind == "grouped_bf16":
        w, factor = v.to(BF16), 1
    else:
        values, scale = v.float().to(orc.F8), torch.full((max(experts, 1), -(-n // 128), -(-k // 128)), 2.0, device="cuda")
        w, factor = ops.f8_pack(values, scale) if experts else ops.f8_pack(values[0], scale[0]), 2
    if not experts:
        assert torch.equal(ops.linear_f8(x, w), (factor * (x.double() @ v[0].double().t())).to(BF16))
        return
    starts = cut_rows(rows, experts, seed=k)
    got = ops.grouped_linear(x, w, starts) if kind == "grouped_bf16" else ops.grouped_linear_f8(x, w, starts)
    want, s = torch.zeros(rows, n, device="cuda", dtype=BF16), starts.tolist()
    for e in range(experts):
        want[s[e] : s[e + 1]] = (factor * (x[s[e] : s[e + 1]].double() @ v[e].double().t())).to(BF16)
    assert torch.equal(got, want)
