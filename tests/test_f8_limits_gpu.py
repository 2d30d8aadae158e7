"""Numbers at the ends of fp32's range in norms and products of 8 bits: what the header says of them."""
import pytest
import torch

import f8_oracle as orc
from test_f8_gpu import BF16, I32, gen, randn, weight
from tinygpt_b200 import ops


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [8, 1000, 20000])
def test_norm_of_rows_past_the_sum_of_squares(built_lib, dim):
    """A row whose squares' sum passes the largest fp32 number reads as zeros, as rms_norm's does; the sum with the residual and the other rows are what they are."""
    x, w = randn(3, dim, seed=1), randn(dim, seed=2)
    x[1, dim // 2], x[1, 0] = 3e19, -1e30
    want = ops.f8_rows_dequantize(ops.rms_norm_f8(x[::2].contiguous(), w, 1e-6))
    back = ops.f8_rows_dequantize(ops.rms_norm_f8(x, w, 1e-6))
    assert not bool(back[1].any()) and not bool(ops.rms_norm(x, w, 1e-6)[1].any()) and torch.equal(back[::2], want)
    rows, z = ops.add_rms_norm_f8(x, torch.zeros_like(x), w, 1e-6)
    assert torch.equal(z, x) and torch.equal(ops.f8_rows_dequantize(rows), back)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3, 200, 300), (100, 264, 1000), (600, 1030, 520)], ids=lambda v: str(v))
@pytest.mark.parametrize("small", [2.0 ** -12, 1e-6])
def test_products_of_small_scales(built_lib, m, n, k, small):
    """A product of scales below the normal numbers is rounded to a multiple of 2^-149: a block's value sum, below 448²·128 < 2^25, is then off by less than 2^-125."""
    x = (randn(m, k, seed=m).float() * 2.0 ** -112).to(BF16)
    rows, w = ops.f8_rows(x), weight(n, k, seed=n)
    w = w._replace(scale=w.scale * small)
    full, held = orc.dense(w), orc.held(rows)
    blocks = -(-k // 128)
    starts = torch.tensor([0, 1, m], device="cuda", dtype=I32)
    both = ops.f8_pack(torch.stack([w.q[:, :k].contiguous()] * 2), torch.stack([w.scale] * 2))
    for y in (ops.linear_f8(rows, w), ops.grouped_linear_f8(rows, both, starts)):
        want, size = held @ full.t(), held.abs() @ full.abs().t()
        # half a step of bf16 — of its least normal number's, too — and the fp32 sums', as f8_oracle.close has them
        bound = want.abs() * 2.0 ** -8 + 2.0 ** -134 + size * ((k + 32) * 2.0 ** -23) + blocks * 2.0 ** -125
        assert bool(((y.double() - want).abs() <= bound).all()) and bool(want.any())
