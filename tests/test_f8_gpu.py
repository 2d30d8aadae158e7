"""Rows and weights of 8 bits (csrc/f8_rows.cu, group_gemm.cu) against their definitions in 64 bits: layouts, sizes off the blocks of 128 and the tiles, numbers that are
none, refusals, captures and streams."""
import pytest
import torch

import f8_oracle as orc
from tinygpt_b200 import ops
from tinygpt_b200._lib import B200Error

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
SIZES = (1, 7, 8, 100, 127, 128, 129, 136, 896, 1000, 2056, 4096)


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def randn(*shape, seed=0, device="cuda", spread=True):
    g = gen(seed, device)
    x = torch.randn(*shape, generator=g, device=device)
    if spread:
        x = x * torch.exp(torch.randn(shape[-1], generator=g, device=device))
    return x.to(BF16)


def weight(n, k, experts=None, seed=0, device="cuda"):
    g = gen(seed, device)
    lead = () if experts is None else (experts,)
    values = (torch.randn(*lead, n, k, generator=g, device=device) * 110).clamp(-448, 448).to(orc.F8)
    scale = torch.exp(torch.randn(*lead, -(-n // 128), -(-k // 128), generator=g, device=device)) / 100
    return ops.f8_pack(values, scale)


def same_rows(got, t, factor=None, rel=0.0):
    """Values bit for bit, scales within rel, zeros behind the rows."""
    values, s = orc.eight(t)
    q = got.q.reshape(-1, got.q.shape[-1])
    assert torch.equal(q[:, : got.k].double(), values) and not bool(q[:, got.k :].view(torch.uint8).any())
    want = s.double() if factor is None else s.double() * factor
    assert bool(((got.scale.t().double() - want).abs() <= want * rel).all())


# ------------------------------------------------------------------------------------------------------------------------- without a device
def test_layouts_without_a_device():
    g = gen(1, "cpu")
    for n, k, lead in ((1, 1, ()), (130, 200, ()), (5, 32, (3,)), (128, 136, (2,))):
        values = (torch.randn(*lead, n, k, generator=g) * 100).clamp(-448, 448).to(orc.F8)
        scale = torch.rand(*lead, -(-n // 128), -(-k // 128), generator=g)
        w = ops.f8_pack(values, scale)
        assert w.q.shape == (*lead, n, -(-k // 16) * 16) and not bool(w.q[..., k:].view(torch.uint8).any())
        full = values.double() * scale.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]
        assert torch.equal(orc.dense(w), full) and torch.equal(ops.f8_dequantize(w), full.float())
        x = torch.randn(*lead, n, k, generator=g)
        x[..., 0, 0] = 1e-41
        back = ops.f8_dequantize(ops.f8_quantize(x)).double()
        s = ops.f8_quantize(x).scale.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]
        # half a step of e4m3, and a rounding to fp32 of the quotient and one of the product
        assert bool(((back - x.double()).abs() <= x.double().abs() * (2.0 ** -4 + 2.0 ** -22) + s * 2.0 ** -10).all())
    zero = ops.f8_quantize(torch.zeros(3, 5))
    assert not bool(ops.f8_dequantize(zero).any())


def test_refusals_without_a_device():
    v, s = torch.zeros(130, 200).to(orc.F8), torch.ones(2, 2)
    w = ops.f8_pack(v, s)
    for bad in (lambda: ops.f8_pack(v.float(), s), lambda: ops.f8_pack(v, s[:1]), lambda: ops.f8_pack(v, s.double()), lambda: ops.f8_pack(v[0], s),
                lambda: ops.f8_pack(v[:0], s[:0]), lambda: ops.f8_quantize(torch.full((2, 8), float("nan"))), lambda: ops.f8_quantize(torch.zeros(2, 8).int()),
                lambda: ops.f8_quantize(torch.zeros(8)), lambda: ops.f8_pack(torch.zeros(1025, 1, 16).to(orc.F8), torch.ones(1025, 1, 1))):
        with pytest.raises(B200Error):
            bad()
    x = torch.zeros(2, 200, dtype=BF16)
    three = ops.f8_pack(v[None].contiguous(), s[None].contiguous())
    for call in (lambda: ops.f8_rows(x), lambda: ops.rms_norm_f8(x, None, 1e-6), lambda: ops.add_rms_norm_f8(x, x, None, 1e-6), lambda: ops.silu_mul_f8(x),
                 lambda: ops.linear_f8(x, w), lambda: ops.grouped_linear(x, torch.zeros(1, 4, 200, dtype=BF16), torch.zeros(2, dtype=I32)),
                 lambda: ops.grouped_linear_f8(x, three, torch.zeros(2, dtype=I32)), lambda: ops.expert_order(torch.zeros(2, 1, dtype=I32), 4),
                 lambda: ops.expert_combine(x, torch.zeros(2, 1, dtype=I32), torch.zeros(2, 1))):
        with pytest.raises(B200Error, match="CUDA device"):
            call()


# ---------------------------------------------------------------------------------------------------------------------------------- rows
@pytest.mark.gpu
@pytest.mark.parametrize("k", SIZES)
def test_rows(built_lib, k):
    for rows in (1, 3, 130):
        x = randn(rows, k, seed=k + rows)
        x[0] = 0
        if rows > 2:
            x[1] *= 2.0 ** -120   # blocks whose scale is the least one, or near it
            x[2] *= 2.0 ** 100
        got = ops.f8_rows(x)
        same_rows(got, x.double())
        back = ops.f8_rows_dequantize(got)
        assert back.shape == x.shape and torch.equal(back.double(), orc.held(got).float().double())


@pytest.mark.gpu
def test_rows_from_a_list_and_from_afar(built_lib):
    x = randn(9, 200)
    index = torch.tensor([8, 0, 0, -1, 3, 9, 7, 2 ** 31 - 1, -2 ** 31], device="cuda", dtype=I32)
    got = ops.f8_rows(x, index)
    want = torch.stack([x[i] if 0 <= i < 9 else torch.zeros_like(x[0]) for i in index.tolist()])
    same_rows(got, want.double())
    wide = randn(9, 512)
    for cols in (slice(0, 200), slice(8, 208), slice(3, 203)):
        same_rows(ops.f8_rows(wide[:, cols]), wide[:, cols].double())
        same_rows(ops.f8_rows(wide[:, cols], index), torch.stack([wide[i, cols] if 0 <= i < 9 else 0 * wide[0, cols] for i in index.tolist()]).double())
    same_rows(ops.f8_rows(wide.t()), wide.t().double())
    got = ops.f8_rows(x.view(3, 3, 200))
    assert got.q.shape == (3, 3, 208) and ops.f8_rows_dequantize(got).shape == (3, 3, 200)
    assert ops.f8_rows(x[0]).q.shape == (208,)
    empty = ops.f8_rows(x[:0])
    assert empty.q.shape == (0, 208) and ops.f8_rows_dequantize(empty).shape == (0, 200)
    none = ops.f8_rows(x[:0], index)   # a list into nothing
    assert not bool(ops.f8_rows_dequantize(none).any())


@pytest.mark.gpu
def test_rows_that_are_not_finite(built_lib):
    x = randn(4, 300)
    x[1, 5], x[2, 200], x[3, 299] = float("nan"), float("inf"), -float("inf")
    back = ops.f8_rows_dequantize(ops.f8_rows(x))
    same = ops.f8_rows_dequantize(ops.f8_rows(torch.where(x.isfinite(), x, 0 * x)))
    assert torch.equal(back[0], same[0]) and torch.equal(back[1, 128:], same[1, 128:]) and torch.equal(back[2, :128], same[2, :128])
    assert bool(back[1, 5].isnan()) and bool(back[2, 200].isnan()) and bool(back[3, 299].isnan())
    w = weight(40, 300)
    y = ops.linear_f8(x, w)
    assert bool(y[0].isfinite().all()) and not bool(y[1:].isfinite().any())   # a row's values reach that row alone
    assert torch.equal(y[0], ops.linear_f8(torch.where(x.isfinite(), x, 0 * x), w)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dim", SIZES + (8192, 16384, 20000, 20001))
def test_norms(built_lib, dim):
    eps = 1e-5
    # an entry's square, its chain of sums in a thread (32 entries, or 8 of every 8 192), 5 + 16 levels over the CTA, the mean's two roundings: half of
    # it passes the root; the root's own rounding and the scale's two
    rel = ((max(32, 8 * (-(-dim // 8192))) + 24) / 2 + 3) * 2.0 ** -24
    for rows in (1, 5):
        x, r, w = randn(rows, dim, seed=1), randn(rows, dim, seed=2), (1 + randn(dim, seed=3, spread=False) * 0.25)
        z = (x.double() + r.double()).to(BF16)
        for weight_ in (w, None):
            t = lambda v: v.double() * (1 if weight_ is None else weight_.double())
            inv = lambda v: 1 / (v.double().square().mean(1, keepdim=True) + eps).sqrt()
            same_rows(ops.rms_norm_f8(x, weight_, eps), t(x), inv(x), rel)
            got, total = ops.add_rms_norm_f8(x, r, weight_, eps)
            assert torch.equal(total, z)
            same_rows(got, t(z), inv(z), rel)
    x = randn(2, 3, dim)
    assert torch.equal(ops.rms_norm_f8(x, w, eps).q.view(torch.uint8).view(6, -1), ops.rms_norm_f8(x.view(6, dim), w, eps).q.view(torch.uint8))


@pytest.mark.gpu
def test_norm_of_rows_without_a_number(built_lib):
    x = randn(3, 300)
    x[0], x[1, 7] = 0, float("nan")
    got = ops.f8_rows_dequantize(ops.rms_norm_f8(x, None, 1e-6))
    assert not bool(got[0].any()) and bool(got[1, :128].isnan().any()) and bool(got[1].isnan().any()) and bool(got[2].isfinite().all())
    assert ops.rms_norm_f8(x[:0], None, 1e-6).q.shape == (0, 304)


@pytest.mark.gpu
def test_norm_sums_where_the_row_was(built_lib):
    """The C call may put the sum over the row or the residual, in rows that a CTA holds and in longer ones."""
    from tinygpt_b200._lib import check, lib
    for dim in (1000, 1001, 20000):
        x, r, w = randn(3, dim, seed=1), randn(3, dim, seed=2), randn(dim, seed=3)
        want, total = ops.add_rms_norm_f8(x, r, w, 1e-6)
        for over in (0, 1):
            a = [x.clone(), r.clone()]
            got = ops._f8_empty((3,), dim, x.device)
            check(lib().b200_rmsnorm_f8(got.q.data_ptr(), got.scale.data_ptr(), a[over].data_ptr(), a[0].data_ptr(), a[1].data_ptr(), w.data_ptr(), 3, dim, 1e-6,
                                        torch.cuda.current_stream().cuda_stream))
            assert torch.equal(a[over], total) and torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(got.scale, want.scale)


@pytest.mark.gpu
@pytest.mark.parametrize("n", SIZES)
def test_silu_products(built_lib, n):
    x = randn(37, 2 * n, seed=n)
    x[0] = 0
    got = ops.silu_mul_f8(x)
    g, u = x[:, :n].double(), x[:, n:].double()
    t = g / (1 + torch.exp(-g)) * u
    want = orc.scales(t).double()
    rel = 2.0 ** -20   # exp, sum, quotient and product in fp32: some steps of 2^-23
    assert bool(((got.scale.t().double() - want).abs() <= want * rel + 2.0 ** -126).all())
    # half a step of e4m3, plus the above
    bound = t.abs() * (2.0 ** -4 + 2 * rel) + orc.spread(want, n) * 2.0 ** -10 * (1 + rel)
    assert bool(((orc.held(got) - t).abs() <= bound).all())
    assert not bool(got.q[:, n:].view(torch.uint8).any())
    x[1, 3 % n] = -200.0   # silu → 0, not NaN
    x[2, n] = float("nan")
    back = ops.f8_rows_dequantize(ops.silu_mul_f8(x))
    assert bool(back[1].isfinite().all()) and bool(back[2, 0].isnan())


# ------------------------------------------------------------------------------------------------------------------------------- products
ROWS = (1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 129, 200, 256, 257, 300, 520)


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", [(1, 1), (8, 128), (130, 100), (128, 129), (1000, 1000), (2049, 520), (300, 4100), (4112, 1024), (20000, 200)])
def test_linear(built_lib, n, k):
    w = weight(n, k, seed=n + k)
    full, bias = orc.dense(w), randn(n, seed=5)
    for m in ROWS:
        x = randn(m, k, seed=m)
        rows = ops.f8_rows(x)
        y = ops.linear_f8(rows, w)
        orc.close(y, orc.held(rows), full)
        orc.close(ops.linear_f8(x, w, bias), orc.held(rows), full, bias)
        assert torch.equal(ops.linear_f8(x, w), y)


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,m", [(4096, 14336, 3), (28672, 4096, 1), (4096, 4096, 1111), (1152, 896, 2048), (512, 16384, 700)])
def test_linear_sizes_of_models(built_lib, n, k, m):
    w, x = weight(n, k, seed=1), randn(m, k, seed=2)
    rows = ops.f8_rows(x)
    orc.close(ops.linear_f8(rows, w), orc.held(rows), orc.dense(w))


@pytest.mark.gpu
def test_linear_sums_that_are_exact(built_lib):
    """Whole numbers whose sums fp32 and bf16 hold: every term counts once, whatever the tiles and splits."""
    for n, k, m in ((300, 1000, 1), (300, 1000, 40), (260, 2000, 100), (140, 384, 300), (2000, 500, 530)):
        g = gen(n + m)
        x = torch.zeros(m, k, device="cuda", dtype=BF16)
        x[:, ::7] = torch.randint(-1, 2, (m, len(range(0, k, 7))), generator=g, device="cuda").to(BF16)
        x[:, 0::128] = 448   # the block's scale is 1
        w = ops.f8_pack(torch.randint(-1, 2, (n, k), generator=g, device="cuda").float().to(orc.F8), torch.full((-(-n // 128), -(-k // 128)), 2.0, device="cuda"))
        want = 2 * (x.double() @ w.q[:, :k].double().t())
        got = ops.linear_f8(x, w)
        assert torch.equal(got, want.to(BF16))


def groups(counts, before=0, behind=0):
    s = [before]
    for c in counts:
        s.append(s[-1] + c)
    return torch.tensor(s, device="cuda", dtype=I32), s[-1] + behind


def each_group(y, x, w, starts):
    s = starts.tolist()
    for e in range(len(s) - 1):
        orc.close(y[s[e] : s[e + 1]], x[s[e] : s[e + 1]], w[e])
    assert not bool(y[: s[0]].any()) and not bool(y[s[-1] :].any())


COUNTS = [(0, 1, 300, 17, 0, 64, 129, 5, 0, 33, 2, 256, 90, 1, 0), (0,) * 7 + (1,) + (0,) * 8, (1,) * 40, (0, 0, 700, 0), (5,), (16, 15, 17, 32, 31, 33), (257, 1, 255)]


@pytest.mark.gpu
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("n,k", [(8, 8), (130, 104), (260, 520), (513, 136), (1000, 1032)])
def test_grouped(built_lib, counts, n, k):
    for before, behind in ((0, 0), (3, 11)):
        starts, rows = groups(counts, before, behind)
        x = randn(rows, k, seed=1)
        w = (torch.randn(len(counts), n, k, generator=gen(2), device="cuda") / k ** 0.5).to(BF16)
        each_group(ops.grouped_linear(x, w, starts), x.double(), w.double(), starts)
        w8, x8 = weight(n, k - 3, len(counts), seed=3), ops.f8_rows(x[:, : k - 3])
        y = ops.grouped_linear_f8(x8, w8, starts)
        each_group(y, orc.held(x8), orc.dense(w8), starts)
        assert torch.equal(y, ops.grouped_linear_f8(x[:, : k - 3].contiguous(), w8, starts))


@pytest.mark.gpu
def test_grouped_in_every_tile_size(built_lib):
    """Average groups of 1 to 300 rows take tiles of 16 to 256 rows; one group among them has far more, others none."""
    n, k = 200, 264
    for each, experts in ((1, 30), (8, 20), (20, 12), (50, 8), (200, 5)):
        counts = [(each * (e % 3)) for e in range(experts)]
        counts[2] = 5 * each + 3
        starts, rows = groups(counts)
        x, w = randn(rows, k, seed=each), (torch.randn(experts, n, k, generator=gen(each), device="cuda") / 16).to(BF16)
        each_group(ops.grouped_linear(x, w, starts), x.double(), w.double(), starts)
        w8, x8 = weight(n, k, experts, seed=each), ops.f8_rows(x)
        each_group(ops.grouped_linear_f8(x8, w8, starts), orc.held(x8), orc.dense(w8), starts)


@pytest.mark.gpu
def test_grouped_writes_its_rows_alone(built_lib):
    """Memory around y stays as it was; starts that fall or leave the rows write inside y all the same."""
    from tinygpt_b200._lib import check, lib
    n, k, rows, experts = 130, 72, 40, 4
    x, w = randn(rows, k), randn(experts, n, k, spread=False)
    st = torch.cuda.current_stream().cuda_stream
    for s in ([0, 3, 3, 30, 40], [2, 5, 9, 9, 33], [-7, 10, 20, 30, 90], [0, 30, 10, 40, 35], [40, 0, 0, 0, 0], [2 ** 31 - 1, -2 ** 31, 5, 2 ** 31 - 1, 0]):
        box = torch.full((rows + 64, n), 7.0, device="cuda", dtype=BF16)
        starts = torch.tensor(s, device="cuda", dtype=I32)
        check(lib().b200_grouped_bf16(box[32:].data_ptr(), x.data_ptr(), w.data_ptr(), starts.data_ptr(), rows, experts, n, k, st))
        assert bool((box[:32] == 7).all()) and bool((box[32 + rows :] == 7).all())
        if s == sorted(s) and s[0] >= 0 and s[-1] <= rows:
            each_group(box[32 : 32 + rows], x.double(), w.double(), starts)


@pytest.mark.gpu
def test_products_of_all_kinds_of_calls(built_lib):
    w, x = weight(200, 136), randn(2, 3, 136)
    rows = ops.f8_rows(x)
    y = ops.linear_f8(rows, w)
    assert y.shape == (2, 3, 200)
    orc.close(y.view(6, 200), orc.held(rows), orc.dense(w))
    assert ops.linear_f8(x[0, 0], w).shape == (200,) and ops.linear_f8(x[:0], w).shape == (0, 3, 200)
    assert torch.equal(ops.linear_f8(x.transpose(0, 1), w), y.transpose(0, 1))
    off = torch.empty(rows.q.numel() + 8, device="cuda", dtype=torch.uint8)[8:].view(orc.F8).view(rows.q.shape)   # 8 bytes off the boundary
    off.view(torch.uint8).copy_(rows.q.view(torch.uint8))
    assert torch.equal(ops.linear_f8(rows._replace(q=off), w), y)
    w3, starts = weight(200, 136, 2), torch.tensor([0, 1, 6], device="cuda", dtype=I32)
    assert ops.grouped_linear_f8(x.view(6, 136)[:0], w3, starts).shape == (0, 200)
    bad = [lambda: ops.linear_f8(x.float(), w), lambda: ops.linear_f8(x[..., :128], w), lambda: ops.linear_f8(x, w3), lambda: ops.linear_f8(x, w.q),
           lambda: ops.linear_f8(x, w, torch.zeros(199, device="cuda", dtype=BF16)), lambda: ops.linear_f8(x, w._replace(n=300)), lambda: ops.linear_f8(x.cpu(), w),
           lambda: ops.linear_f8(x, w._replace(k=144)), lambda: ops.linear_f8(x, w._replace(n=2 ** 70)), lambda: ops.linear_f8(rows._replace(k=130), w),
           lambda: ops.linear_f8(rows._replace(scale=rows.scale[:, :5]), w), lambda: ops.grouped_linear_f8(x, w3, starts),
           lambda: ops.grouped_linear_f8(x.view(6, 136), w, starts), lambda: ops.grouped_linear_f8(x.view(6, 136), w3, starts[:2]),
           lambda: ops.grouped_linear_f8(x.view(6, 136), w3, starts.long()), lambda: ops.grouped_linear(x.view(6, 136), randn(2, 5, 128), starts),
           lambda: ops.grouped_linear(randn(6, 12), randn(2, 5, 12), starts), lambda: ops.rms_norm_f8(x, randn(100), 1e-6), lambda: ops.silu_mul_f8(randn(2, 7)),
           lambda: ops.add_rms_norm_f8(x, x[:1], None, 1e-6), lambda: ops.add_rms_norm_f8(x, None, None, 1e-6), lambda: ops.f8_rows(x, starts),
           lambda: ops.f8_rows(x.view(6, 136), starts.long()), lambda: ops.f8_rows_dequantize(rows._replace(k=100))]
    for call in bad:
        with pytest.raises(B200Error):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 100, 300])
def test_captured_and_on_another_stream(built_lib, m):
    w, w3 = weight(200, 264), weight(264, 200, 4)
    x, r, g = randn(m, 264, seed=1), randn(m, 264, seed=2), randn(264, seed=3)
    starts, other = (torch.tensor(s, device="cuda", dtype=I32) for s in ([0, 1, 1, m // 2, m], [0, 0, m - 1, m - 1, m]))

    def chain(x, starts):
        rows, z = ops.add_rms_norm_f8(x, r, g, 1e-6)
        y = ops.linear_f8(rows, w)
        return ops.grouped_linear_f8(y, w3, starts) + z

    want = [chain(x, starts), chain(x.flip(0), other)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        assert torch.equal(chain(x, starts), want[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = chain(x, starts)
        graph.replay()
        st.synchronize()
        assert torch.equal(out, want[0])
        x.copy_(x.flip(0))
        starts.copy_(other)
        graph.replay()
    st.synchronize()
    assert torch.equal(out, want[1])
