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
