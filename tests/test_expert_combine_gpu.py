"""expert_combine next to numbers that are none: what no place names counts nothing, what one names reaches its own row alone."""
import pytest
import torch

from test_f8_gpu import I32, gen, randn
from tinygpt_b200 import ops


@pytest.mark.gpu
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("n", [1, 100, 200, 2056])
@pytest.mark.parametrize("rows,top", [(5, 4), (300, 2), (40, 9)])
def test_rows_that_are_not_finite(built_lib, rows, top, n, what):
    pairs, g = rows * top, gen(rows)
    y, w = randn(pairs, n, seed=n), torch.rand(rows, top, generator=g, device="cuda") + 0.5
    place = torch.randperm(pairs, generator=g, device="cuda").to(I32).view(rows, top)
    used = int(place[-1, 0])   # a row of y that the last row takes
    place[0, 0], place[1, top - 1], place[2, 0], place[3, 0] = -1, pairs, 2 ** 31 - 1, -2 ** 31
    free = sorted(set(range(pairs)) - set(place.flatten().tolist()))   # rows of y that no place names
    clean = ops.expert_combine(y, place, w)
    bad = y.clone()
    bad[free] = what
    assert torch.equal(ops.expert_combine(bad, place, w), clean)
    bad[used, n // 2] = what
    got = ops.expert_combine(bad, place, w)
    assert not bool(got[-1, n // 2].isfinite())
    got[-1, n // 2] = clean[-1, n // 2]
    assert torch.equal(got, clean)
    # a weight beside a place that is none counts nothing, either
    w[0, 0], w[1, top - 1], w[2, 0], w[3, 0] = what, -what, what, what
    assert torch.equal(ops.expert_combine(y, place, w), clean)
    # nothing chosen at all: zeros, whatever lies in y
    none = ops.expert_combine(torch.full_like(y, what), torch.full_like(place, -1), w)
    assert not bool(none.any())
