"""Parts of 8-bit weights as a user's program may hold them."""
import pytest
import torch

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
