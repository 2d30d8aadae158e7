"""Weights of 4 bits where they can go wrong: matrices next to the largest number, values and sizes of more bits than a layout holds."""
import pytest
import torch

from tinygpt_b200 import ops
from tinygpt_b200._lib import B200Error


def unpacked(w):
    """W of a W4Weight, in 64 bits (CPU)."""
    tiles, blocks, groups = -(-w.n // 16), -(-w.k // 64), -(-w.k // w.group)
    v = torch.stack((w.q & 15, w.q >> 4), -1).view(tiles, blocks, 8, 4, 2, 2, 2, 2, 2).permute(0, 8, 2, 1, 4, 3, 5, 7, 6).reshape(tiles * 16, blocks * 64)[:w.n, :w.k]
    back = lambda t: t.permute(0, 3, 2, 1).reshape(-1, groups)[:w.n].double().repeat_interleave(w.group, 1)[:, :w.k]
    return back(w.scale) * (v.double() - (8 if w.zero is None else back(w.zero))), back(w.scale)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 128])
def test_quantize_to_the_ends_of_fp32(symmetric, group):
    """A group's range may pass the largest fp32 number though its entries do not."""
    g = torch.Generator().manual_seed(5)
    w = (torch.rand(4, 200, generator=g) * 2 - 1) * 3e38
    w[1, :7] = 3.3e38
    w[2] = w[2].abs()
    w[3] = -w[3].abs()
    got, s = unpacked(ops.w4_quantize(w, group=group, symmetric=symmetric))
    assert bool(torch.isfinite(got).all())
    # half a step; the range's ends lose what the scale's rounding (2^-8 of up to 15 steps) and the zero's to a whole number take: half a step more
    assert bool(((got - w.double()).abs() <= s * (0.5 + 15 * 2.0 ** -8 + (0 if symmetric else 0.5))).all())


def test_pack_refuses_values_of_more_bits():
    v, s = torch.full((16, 64), 15, dtype=torch.uint8), torch.ones(16, 1).to(torch.bfloat16)
    assert bool((ops.w4_pack(v, s).q == 255).all())
    for bad in (16, 255):
        v[15, 63] = bad
        with pytest.raises(B200Error, match="0 … 15"):
            ops.w4_pack(v, s)


def test_sizes_that_a_descriptor_does_not_hold_are_refused():
    """n, k and the group reach the library in 32 bits; a W4Weight made by hand may hold more, which must not come out as others."""
    w = ops.w4_pack(torch.zeros(16, 128, dtype=torch.uint8), torch.ones(16, 1).to(torch.bfloat16), group=128)
    for bad, what in ((w._replace(group=2 ** 32 + 64), "groups of"), (w._replace(group=48), "groups of"), (w._replace(group=0), "groups of"),
                      (w._replace(n=2 ** 32 + 16), "out of range"), (w._replace(k=2 ** 32 + 128), "out of range"), (w._replace(k=-128), "out of range"),
                      (w._replace(n=0), "out of range")):
        for call in (ops.w4_dequantize, lambda w: ops.linear_w4(torch.zeros(1, 128, dtype=torch.bfloat16), w)):
            with pytest.raises(B200Error, match=what):
                call(bad)


@pytest.mark.gpu
def test_sizes_that_a_descriptor_does_not_hold_are_refused_on_the_device(built_lib):
    w = ops.w4_pack(torch.zeros(16, 128, dtype=torch.uint8, device="cuda"), torch.ones(16, 1, device="cuda").to(torch.bfloat16), group=128)
    x = torch.ones(3, 128, device="cuda", dtype=torch.bfloat16)
    assert bool((ops.linear_w4(x, w) == -8 * 128).all())
    for bad in (w._replace(group=2 ** 32 + 64), w._replace(group=2 ** 32 + 128), w._replace(n=2 ** 32 + 16), w._replace(k=2 ** 32 + 128)):
        for call in (lambda: ops.linear_w4(x, bad), lambda: ops.w4_dequantize(bad)):
            with pytest.raises(B200Error):
                call()


@pytest.mark.gpu
@pytest.mark.parametrize("group,zero", [(32, None), (64, 128.0), (128, None), (128, 128.0), (128, -128.0), (128, 7.5)])
@pytest.mark.parametrize("m", [1, 8, 20, 60, 100, 300])
def test_inputs_up_to_the_stated_bound(built_lib, m, group, zero):
    """Entries of x of one sign just below 2^112: the sums in front of a group's scale are as large as they come, the result is not."""
    n, k = 264, 520
    g = torch.Generator(device="cuda").manual_seed(7)
    v = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    v[:8], v[8:16] = 15, 8
    s = ((torch.rand(n, -(-k // group), generator=g, device="cuda") + 0.5) * 2.0 ** -10).to(torch.bfloat16)
    z = None if zero is None else torch.full_like(s, zero)
    x = ((1 - torch.rand(m, k, generator=g, device="cuda") * 0.25) * 2.0 ** 112).to(torch.bfloat16).clamp(max=2.0 ** 112 * (1 - 2.0 ** -8))
    x[m // 2] = -x[m // 2]
    y = ops.linear_w4(x, ops.w4_pack(v, s, z, group=group)).double()
    full = s.double().repeat_interleave(group, 1)[:, :k] * (v.double() - (8 if zero is None else zero))
    # half a step of the result; fp32 sums of k terms, each no more than (128 + 15 + |zero|) scales; beyond the exact way a weight's rounding
    size = x.double().abs() @ (s.double().repeat_interleave(group, 1)[:, :k] * (143 + abs(zero or 8))).t()
    bound = (x.double() @ full.t()).abs() * 2.0 ** -8 + size * k * 2.0 ** -23 + (x.double().abs() @ full.abs().t() * 2.0 ** -9 if m > 64 else 0)
    assert bool(torch.isfinite(y).all()) and bool(((y - x.double() @ full.t()).abs() <= bound).all())


# ------------------------------------------------------------------------------------------------- sums that are exact
def whole_numbers(n, k, group, zero, seed=9, device="cuda"):
    """A weight of values times powers of two from 1/2 to 2, zeros whole and halves: exact as bf16, and so is every sum over it of whole numbers x in fp32 (8 200 columns of
    at most 3·(128 + 15)·2, and 3·(128 + 15)·2 beside them for the zeros, in halves: below 2^24 by far, and so in every order)."""
    g = torch.Generator(device=device).manual_seed(seed)
    v = torch.randint(0, 16, (n, k), generator=g, device=device, dtype=torch.uint8)
    shape = (n, -(-k // group))
    s = torch.exp2(torch.randint(-1, 2, shape, generator=g, device=device).float()).to(torch.bfloat16)
    z = None
    if zero:
        z = torch.randint(0, 16, shape, generator=g, device=device).float()
        z[n // 2:] += 0.5 * torch.randint(0, 2, (n - n // 2, shape[1]), generator=g, device=device)
        z = z.to(torch.bfloat16)
    full = s.double().repeat_interleave(group, 1)[:, :k] * (v.double() - (8 if z is None else z.double().repeat_interleave(group, 1)[:, :k]))
    return ops.w4_pack(v, s, z, group=group), full, g


def rows_of(m, k, g):
    return torch.randint(-3, 4, (m, k), generator=g, device=g.device).to(torch.bfloat16)


SIZES = [(1032, 8200), (24, 4096), (4104, 2056), (8200, 1000), (20008, 512), (28672, 264), (999, 520), (40, 8)]


@pytest.mark.parametrize("n,k", [(1032, 8200), (24, 4096), (200, 2056)])
@pytest.mark.parametrize("zero", [False, True])
def test_no_lost_columns_pass(n, k, zero):
    """Eight columns, a stage of 128 or the share of one of eight CTAs, lost or counted twice, move results that have to be equal, of every row."""
    _, full, g = whole_numbers(n, k, 64, zero, device="cpu")
    x = rows_of(40, k, g).double()
    want = (x @ full.t()).to(torch.bfloat16)
    for first, many in ((0, 8), (k - 8, 8), (0, 128), (k // 256 * 128, 128), (k - k % 128 if k % 128 else k - 128, 128), (k // 8 * 3, k // 8)):
        lost = x.clone()
        lost[:, first:first + many] = 0
        for bad in (lost, 2 * x - lost):
            assert bool(((bad @ full.t()).to(torch.bfloat16) != want).any(1).all()), (first, many)


@pytest.mark.gpu
@pytest.mark.parametrize("group,zero", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("n,k", SIZES)
def test_whole_numbers_are_exact(built_lib, n, k, group, zero):
    """Every way, at every number of rows around its ends: nothing but the result is rounded, so that every column counts once."""
    w, full, g = whole_numbers(n, k, group, zero)
    bias = torch.randint(-64, 65, (n,), generator=g, device="cuda").to(torch.bfloat16)
    assert torch.equal(ops.w4_dequantize(w).double(), full)
    for m in (1, 2, 8, 9, 16, 17, 24, 32, 33, 40, 64, 65, 80, 100, 128, 129, 200, 256, 257, 300):
        x = rows_of(m, k, g)
        want = x.double() @ full.t()
        assert torch.equal(ops.linear_w4(x, w), want.to(torch.bfloat16)), m
        assert torch.equal(ops.linear_w4(x, w, bias), (want + bias.double()).to(torch.bfloat16)), m


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,m", [(24, 72, 1), (4104, 520, 20), (999, 520, 70), (264, 1096, 60), (4104, 520, 129), (1032, 72, 300)])
def test_calls_of_the_library_stay_within_their_memory(built_lib, n, k, m):
    """The C entry points with a workspace and results of just the bytes they ask for, whatever those held before."""
    import ctypes as C
    from test_kv4_edges_gpu import Guarded
    from tinygpt_b200._lib import W4Desc, lib
    w, full, g = whole_numbers(n, k, 64, True)
    x, bias, stream = rows_of(m, k, g), torch.randint(-64, 65, (n,), generator=g, device="cuda").to(torch.bfloat16), torch.cuda.current_stream().cuda_stream
    d = W4Desc(w.q.data_ptr(), w.scale.data_ptr(), w.zero.data_ptr(), n, k, 64)
    for b in (None, bias):
        y, ws = Guarded(2 * m * n), Guarded(lib().b200_w4_workspace_bytes(m, n, k))
        assert lib().b200_w4_linear_bf16(y.at, x.data_ptr(), C.byref(d), None if b is None else b.data_ptr(), m, ws.at if ws.nbytes else None, stream) == 0
        want = x.double() @ full.t() + (0 if b is None else b.double())
        assert torch.equal(y.view(torch.bfloat16, m, n), want.to(torch.bfloat16)) and y.intact() and ws.intact()
    out = Guarded(2 * n * k)
    assert lib().b200_w4_dequant_bf16(out.at, C.byref(d), stream) == 0
    assert torch.equal(out.view(torch.bfloat16, n, k).double(), full) and out.intact()
