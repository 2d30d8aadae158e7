"""silu_mul_f8 over every gate that bf16 has, the largest and the least, infinities and NaN among them."""
import pytest
import torch

import f8_oracle as orc
from test_f8_gpu import BF16, I32, gen, weight
from tinygpt_b200 import ops


def every_finite():
    bits = torch.arange(-32768, 32768, device="cuda", dtype=I32).to(torch.int16)
    x = bits.view(BF16)
    return x[x.isfinite()]


# fp32 steps behind gate and up: exp2 2^-22, reciprocal 2^-23, four roundings of 2^-24 (the exponential's correction, the sum, two products) and the scale's — below 2^-20.
# A silu below 2^-119 may be 0.  A block's scale is at least 2^-126, so that entries below 448·2^-126 are off by half a step of e4m3, and of its least step.
def bound(silu, up):
    t = silu * up
    tiny = t.abs() < 450 * 2.0 ** -126
    return t.abs() * 2.0 ** -20 + tiny * (t.abs() * 2.0 ** -4 + 2.0 ** -136 * 1.01) + up.abs() * silu.abs() * (silu.abs() < 2.0 ** -119 * 1.0001)


def silu_of(gate):
    g = gate.double()
    return g * torch.special.expit(g)


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("up", [1.0, -1.0, 0.5, 0.0])
def test_every_gate_by_itself(built_lib, up, wide):
    """A gate to a block: its scale and its value are its own.  wide: with seven gates of 0 behind it, the rows that are read in pieces of 16 bytes."""
    gate = every_finite()
    x = torch.zeros(len(gate), 16 if wide else 2, device="cuda", dtype=BF16)
    x[:, 0], x[:, x.shape[1] // 2] = gate, up
    got = orc.held(ops.silu_mul_f8(x))
    silu = silu_of(gate)
    assert bool(got.isfinite().all())
    assert bool(((got[:, 0] - silu * up).abs() <= bound(silu, torch.full_like(silu, up))).all())
    assert not bool(got[:, 1:].any())


@pytest.mark.gpu
def test_large_gates_beside_small_ones(built_lib):
    """A large gate with a small up leaves the block's other entries as they are; in experts_f8 and the Linear behind it no row is spoiled."""
    n = 136
    x = torch.randn(6, 2 * n, generator=gen(1), device="cuda").to(BF16)
    want = ops.silu_mul_f8(x)
    for g in (2.3e38, 2.4e38, 3.3e38, -2.4e38, -3.3e38):
        y = x.clone()
        y[2, 5], y[2, n + 5] = g, 0.0
        y[3, 130], y[3, n + 130] = g, 2.0 ** -126
        got = ops.silu_mul_f8(y)
        held = orc.held(got)
        assert bool(held.isfinite().all()) and float(held[2, 5]) == 0
        silu = silu_of(y[3, 130])
        # half a step of e4m3 of the entry or of its block's least step
        assert abs(float(held[3, 130] - silu * 2.0 ** -126)) <= float((silu * 2.0 ** -126).abs() * (2.0 ** -4 + 2.0 ** -19) + got.scale[1, 3].double() * 2.0 ** -10)
        rest = torch.ones(6, n, dtype=torch.bool, device="cuda")
        rest[2, :128] = rest[3, 128:] = False
        assert torch.equal(held[rest], orc.held(want)[rest])
        assert bool(ops.linear_f8(got, weight(40, n)).isfinite().all())


@pytest.mark.gpu
def test_gates_that_are_not_finite(built_lib):
    """silu(∞)·up is ∞ or NaN and reads as NaN, and so does what −∞ and NaN give; other rows stay as they were."""
    n = 8
    for g in (float("inf"), -float("inf"), float("nan")):
        for up in (1.0, -1.0, 0.5, 0.0):
            x = torch.randn(3, 2 * n, generator=gen(2), device="cuda").to(BF16)
            same = ops.f8_rows_dequantize(ops.silu_mul_f8(x))
            x[1, 3], x[1, n + 3] = g, up
            back = ops.f8_rows_dequantize(ops.silu_mul_f8(x))
            assert bool(back[1, 3].isnan()) and torch.equal(back[0], same[0]) and torch.equal(back[2], same[2])
