"""Linears over weights of 4 bits (csrc/w4.cu) against the definition in 64 bits: every group size, with and without zeros, row counts around every change of
kernel, sizes off the tiles of 16 × 64, the refusals, capture and other streams."""
import pytest
import torch

from tinygpt_b200 import ops
from tinygpt_b200._lib import B200Error

BF16 = torch.bfloat16


def parts(n, k, group, zero, device="cuda", seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    values = torch.randint(0, 16, (n, k), generator=g, device=device, dtype=torch.uint8)
    groups = -(-k // group)
    scale = (torch.rand(n, groups, generator=g, device=device) * 0.05 + 0.01).to(BF16)
    z = (torch.rand(n, groups, generator=g, device=device) * 15).to(BF16) if zero else None   # between the whole numbers too
    return values, scale, z


def dense(values, scale, zero, group):
    k = values.shape[1]
    s = scale.double().repeat_interleave(group, 1)[:, :k]
    return s * (values.double() - (8 if zero is None else zero.double().repeat_interleave(group, 1)[:, :k]))


def close(got, x, w, bias=None, weight_eps=0.0):
    """|error| ≤ half a step of bf16 of the result + the sums' own: fp32 over k terms (each product exact; no more than a rounding a term, of the
    terms' sum of magnitudes: with a zero the values' and the zero's part are summed apart, each up to 15 steps) + weights as bf16."""
    want = x.double() @ w.t()
    size = x.double().abs() @ (w.abs() + 2 * w.abs().amax()).t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    bound = want.abs() * 2.0 ** -8 + size * (x.shape[-1] * 2.0 ** -23 + weight_eps) + 1e-30
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound).max())


def test_layout_and_refusals_without_a_device():
    v, s, z = parts(19, 72, 32, True, "cpu")
    w = ops.w4_pack(v, s, z, group=32)
    tile = w.q.view(2, 2, 512)
    for n, k in ((0, 0), (7, 71), (8, 3), (15, 40), (18, 65)):
        t, i, b, j = n // 16, n % 16, k // 64, k % 64
        h, c, t4, p, e = j // 32, j % 32 // 8, j % 8 // 4, j % 4 // 2, j % 2
        byte = int(tile[t, b, 16 * (4 * (i % 8) + c) + 4 * (2 * h + t4) + 2 * e + p])
        assert (byte >> 4 if i >= 8 else byte & 15) == int(v[n, k])
        assert float(w.scale[t, k // 32, i % 8, i // 8]) == float(s[n, k // 32]) and float(w.zero[t, k // 32, i % 8, i // 8]) == float(z[n, k // 32])
    for bad in (lambda: ops.w4_pack(v.int(), s, z, group=32), lambda: ops.w4_pack(v, s, z, group=48), lambda: ops.w4_pack(v[:, :68], s, z, group=32),
                lambda: ops.w4_pack(v, s[:, :2], z, group=32), lambda: ops.w4_pack(v, s.float(), z, group=32), lambda: ops.w4_quantize(v),
                lambda: ops.w4_quantize(torch.full((2, 8), float("nan"))), lambda: ops.w4_quantize(torch.zeros(2, 8), group=16)):
        with pytest.raises(B200Error):
            bad()
    x = torch.zeros(1, 72, dtype=BF16)
    for call in (lambda: ops.linear_w4(x, w), lambda: ops.w4_dequantize(w)):
        with pytest.raises(B200Error, match="CUDA device"):
            call()


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 128])
def test_quantize_is_within_half_a_step(symmetric, group):
    g = torch.Generator().manual_seed(3)
    w = torch.randn(20, 200, generator=g)
    w[3] = 0
    w[4] += 5
    q = ops.w4_quantize(w, group=group, symmetric=symmetric)
    n, k = w.shape
    groups = -(-k // group)
    back = lambda t: t.permute(0, 3, 2, 1).reshape(-1, groups)[:n].double().repeat_interleave(group, 1)[:, :k]
    v = torch.stack((q.q & 15, q.q >> 4), -1).view(2, 4, 8, 4, 2, 2, 2, 2, 2).permute(0, 8, 2, 1, 4, 3, 5, 7, 6).reshape(32, 256)[:n, :k]
    s = back(q.scale)
    got = s * (v.double() - (8 if symmetric else back(q.zero)))
    # half a step; the range's ends lose what the scale's rounding (2^-8 of up to 15 steps) and the zero's to a whole number take: half a step more
    assert bool(((got - w.double()).abs() <= s * (0.5 + 15 * 2.0 ** -8 + (0 if symmetric else 0.5)) + 1e-12).all())


@pytest.mark.gpu
@pytest.mark.parametrize("group,zero", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("n,k", [(1, 8), (16, 64), (40, 200), (33, 1000), (264, 1096), (4104, 328), (8200, 264)])
def test_linear_w4(built_lib, n, k, group, zero):
    v, s, z = parts(n, k, group, zero)
    w, full = ops.w4_pack(v, s, z, group=group), dense(v, s, z, group)
    g = torch.Generator(device="cuda").manual_seed(1)
    for m in (1, 7, 8, 9, 16, 17, 32, 33, 64, 65, 100):
        x, b = torch.randn(m, k, generator=g, device="cuda").to(BF16), torch.randn(n, generator=g, device="cuda").to(BF16)
        eps = 2.0 ** -8 if m > 64 and n % 8 == 0 else 0.0
        close(ops.linear_w4(x, w), x, full, None, eps)
        close(ops.linear_w4(x, w, b), x, full, b, eps)
    back = ops.w4_dequantize(w)
    assert torch.equal(back, full.float().to(BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("group,zero", [(32, False), (32, True), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("n,k", [(1032, 8200), (4104, 2056), (8200, 1000), (20008, 512), (24, 4096), (1000, 136), (24, 8)])
def test_many_rows(built_lib, n, k, group, zero):
    """From 33 rows over large weights and 65 over all: tiles of 128 channels that one to eight CTAs share, zeros between the whole numbers and on them, rows past a
    tile's and past what is unpacked into the products."""
    v, s, z = parts(n, k, group, zero)
    g = torch.Generator(device="cuda").manual_seed(2)
    if zero:
        z[: n // 2] = z[: n // 2].round()
    w, full = ops.w4_pack(v, s, z, group=group), dense(v, s, z, group)
    for m in (40, 65, 80, 128, 129, 256, 257):
        x, b = torch.randn(m, k, generator=g, device="cuda").to(BF16), torch.randn(n, generator=g, device="cuda").to(BF16)
        y = ops.linear_w4(x, w)
        close(y, x, full, None, 2.0 ** -8 if m > 64 or n * k > 6_000_000 else 0.0)
        close(ops.linear_w4(x, w, b), x, full, b, 2.0 ** -8 if m > 64 or n * k > 6_000_000 else 0.0)
        x[3, k - 1] = float("inf")
        got = ops.linear_w4(x, w)
        assert not bool(got[3].isfinite().any()) and torch.equal(got[:3], y[:3]) and torch.equal(got[4:], y[4:])   # a row's values reach that row alone


@pytest.mark.gpu
def test_calls_of_all_kinds(built_lib):
    v, s, z = parts(48, 128, 64, True)
    w, full = ops.w4_pack(v, s, z), dense(v, s, z, 64)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, 3, 128, generator=g, device="cuda").to(BF16)
    y = ops.linear_w4(x, w)
    assert y.shape == (2, 3, 48) and torch.equal(y, ops.linear_w4(x, w))
    close(y.view(6, 48), x.view(6, 128), full)
    assert ops.linear_w4(x[0, 0], w).shape == (48,) and ops.linear_w4(x[:0], w).shape == (0, 3, 48)
    wide = torch.randn(5, 256, generator=g, device="cuda").to(BF16)
    assert torch.equal(ops.linear_w4(wide[:, 64:192], w), ops.linear_w4(wide[:, 64:192].contiguous(), w))
    nan = x.clone()
    nan[0, 0, 5] = float("nan")
    got = ops.linear_w4(nan, w).view(6, 48)
    assert bool(got[0].isnan().all()) and torch.equal(got[1:], y.view(6, 48)[1:])   # a row's values reach that row alone
    for m in (6, 100):   # a captured call, replayed on new inputs, on another stream
        rows = torch.randn(m, 128, generator=g, device="cuda").to(BF16)
        want = ops.linear_w4(rows.flip(0), w)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                out = ops.linear_w4(rows, w)
            rows.copy_(rows.flip(0))
            graph.replay()
        st.synchronize()
        assert torch.equal(out, want)
    for bad in (lambda: ops.linear_w4(x.float(), w), lambda: ops.linear_w4(x[..., :64], w), lambda: ops.linear_w4(x, v), lambda: ops.linear_w4(x.cpu(), w),
                lambda: ops.linear_w4(x, w, torch.zeros(47, device="cuda", dtype=BF16)), lambda: ops.linear_w4(x, w._replace(n=64)),
                lambda: ops.linear_w4(x, w._replace(q=w.q[:512])), lambda: ops.linear_w4(x, w._replace(group=48)), lambda: ops.linear_w4(x, w._replace(n=2 ** 70)),
                lambda: ops.linear_w4(torch.zeros(129, device="cuda", dtype=BF16)[1:], w)):
        with pytest.raises(B200Error):
            bad()
