"""Products over bf16 rows read their bias and groups before they wait for the rows: what they read has to be what the calls in front have written."""
import pytest
import torch

from test_f8_gpu import BF16, I32, randn, weight
from tinygpt_b200 import ops


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 1152, 896), (1, 130, 4100), (9, 2000, 4864), (48, 1024, 2048), (100, 520, 304), (700, 1030, 1024)], ids=lambda v: str(v))
def test_a_bias_written_in_front(built_lib, m, n, k):
    """By a copy and by an operator that lets the next one start early, at the same address every time, other rows between; no synchronisation."""
    from tinygpt_b200._lib import check, lib
    w, xs = weight(n, k, seed=1), [randn(m, k, seed=50 + i) for i in range(6)]
    made, zero, now = [randn(n, seed=80 + i) * 64 for i in range(6)], torch.zeros(n, device="cuda", dtype=BF16), torch.empty(n, device="cuda", dtype=BF16)
    want = []
    for x, b in zip(xs, made):
        torch.cuda.synchronize()
        want.append(ops.linear_f8(ops.f8_rows(x), w, b))
        torch.cuda.synchronize()
    st, got = torch.cuda.current_stream().cuda_stream, []
    for _ in range(4):
        for x, b in zip(xs, made):
            now.copy_(b)
            got.append(ops.linear_f8(x, w, now))
        for x, b in zip(xs, made):
            check(lib().b200_add_bf16(now.data_ptr(), b.data_ptr(), zero.data_ptr(), n, st))
            got.append(ops.linear_f8(x, w, now))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % len(want)]), i


@pytest.mark.gpu
@pytest.mark.parametrize("experts", [3, 40, 700])
def test_groups_written_in_front_at_one_address(built_lib, experts):
    """starts copied into one buffer right before the call, other groups every time."""
    rows, n, k = 60, 264, 520
    w, x = weight(n, k, experts, seed=3), randn(rows, k, seed=4)
    rows8 = ops.f8_rows(x)
    cuts = [torch.sort(torch.randint(0, rows + 1, (experts + 1,), generator=torch.Generator().manual_seed(i)))[0].to(I32).cuda() for i in range(8)]
    want = []
    for c in cuts:
        torch.cuda.synchronize()
        want.append(ops.grouped_linear_f8(rows8, w, c))
        torch.cuda.synchronize()
    now, got = cuts[0].clone(), []
    for c in cuts * 3:
        now.copy_(c)
        got.append(ops.grouped_linear_f8(x, w, now))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % len(want)]), i
