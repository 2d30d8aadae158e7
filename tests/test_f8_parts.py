"""Parts of 8-bit weights as a user's program may hold them: made from parameters that take gradients, lying off the 16-byte boundary."""
import pytest
import torch

import f8_oracle as orc
from test_f8_gpu import I32, gen, randn, weight
from tinygpt_b200 import ops


@pytest.mark.parametrize("shape", [(130, 200), (3, 5, 32)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_weight_of_a_parameter_keeps_no_graph(shape, dtype):
    """A parameter's 8-bit weight is a constant: nothing in it holds the 32-bit copies that it was made from."""
    p = torch.nn.Parameter(torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(dtype))
    got, want = ops.f8_quantize(p), ops.f8_quantize(p.detach())
    for a, b in ((got.q, want.q), (got.scale, want.scale)):
        assert not a.requires_grad and a.grad_fn is None and torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert not ops.f8_dequantize(got).requires_grad
    scale = torch.nn.Parameter(want.scale.clone())
    packed = ops.f8_pack(want.q[..., : shape[-1]].contiguous(), scale)
    assert not packed.scale.requires_grad and torch.equal(packed.scale, want.scale)


def off(t, by):
    """t `by` bytes behind a 16-byte boundary"""
    room = torch.empty(t.numel() * t.element_size() + 32, device=t.device, dtype=torch.uint8)
    out = room[by : by + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
    out.view(torch.uint8).copy_(t.view(torch.uint8))
    assert out.data_ptr() % 16 == by and out.is_contiguous()
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("by", [1, 8])
def test_weights_off_the_boundary(built_lib, by):
    """A view of a weight's bytes, as a file that is read as a whole gives it: laid out anew for the call, as rows off the boundary are."""
    x, w, w3 = randn(6, 136), weight(200, 136), weight(264, 136, 4)
    moved, moved3 = w._replace(q=off(w.q, by)), w3._replace(q=off(w3.q, by))
    starts = torch.tensor([0, 1, 1, 4, 6], device="cuda", dtype=I32)
    rows = ops.f8_rows(x)
    for xs in (x, rows, rows._replace(q=off(rows.q, by))):
        assert torch.equal(ops.linear_f8(xs, moved), ops.linear_f8(rows, w))
        assert torch.equal(ops.grouped_linear_f8(xs, moved3, starts), ops.grouped_linear_f8(rows, w3, starts))
    assert torch.equal(ops.f8_dequantize(moved), ops.f8_dequantize(w))
    w_out = weight(136, 132, 4, seed=2)
    chosen = torch.tensor([[0, 3], [1, 2], [2, 2], [3, 0], [-1, 1], [0, 1]], device="cuda", dtype=I32)
    weights = torch.rand(6, 2, generator=gen(1), device="cuda")
    want = ops.experts_f8(x, chosen, weights, w3, w_out)
    assert torch.equal(ops.experts_f8(x, chosen, weights, moved3, w_out._replace(q=off(w_out.q, by))), want)
    orc.close(ops.linear_f8(rows, moved), orc.held(rows), orc.dense(w))
