"""Products over bf16 rows begin to read their weight while the rows are made: what they read has to be what was written in front of them, by whichever call."""
import ctypes as C

import pytest
import torch

from test_f8_gpu import BF16, I32, gen, randn, weight
from tinygpt_b200 import ops
from tinygpt_b200._lib import B200Error


def _stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 1152, 896), (9, 2000, 4864), (48, 1024, 2048), (100, 520, 304), (700, 1030, 1024)], ids=lambda v: str(v))
def test_a_weight_written_in_front(built_lib, m, n, k):
    """Its bytes by a copy and by f8_rows, a kernel that lets the next one start early; no synchronisation between."""
    from tinygpt_b200._lib import check, lib
    assert k % 16 == 0
    ws, xs = [weight(n, k, seed=i) for i in range(6)], [randn(m, k, seed=50 + i) for i in range(6)]
    raw = [randn(n, k, seed=20 + i) for i in range(6)]
    made = [ops.f8_rows(r).q for r in raw]
    now = ops.F8Weight(torch.empty_like(ws[0].q), ws[0].scale.clone(), n, k)
    junk = torch.empty(-(-k // 128), n, device="cuda")
    want = []
    for w, q, x in zip(ws, made, xs):
        rows = ops.f8_rows(x)
        torch.cuda.synchronize()
        want += [ops.linear_f8(rows, w._replace(scale=now.scale)), ops.linear_f8(rows, now._replace(q=q))]
        torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for w, r, x in zip(ws, raw, xs):
            now.q.view(torch.uint8).copy_(w.q.view(torch.uint8))
            got.append(ops.linear_f8(x, now))
            check(lib().b200_f8_rows_bf16(now.q.data_ptr(), junk.data_ptr(), r.data_ptr(), k, n, None, n, k, _stream()))
            got.append(ops.linear_f8(x, now))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % len(want)]), i


@pytest.mark.gpu
@pytest.mark.parametrize("rows,top,experts,n,k", [(4, 2, 8, 264, 520), (60, 4, 32, 512, 1024), (700, 2, 4, 260, 256), (3, 1, 900, 72, 136)], ids=lambda v: str(v))
def test_groups_made_in_front(built_lib, rows, top, experts, n, k):
    """starts by expert_order directly in front, other choices every time; behind it the same, captured and replayed."""
    w = weight(n, k, experts, seed=3)
    x = randn(rows * top, k, seed=4)
    choices = [torch.randint(-1, experts, (rows, top), generator=gen(i), device="cuda", dtype=I32) for i in range(8)]
    rows8 = ops.f8_rows(x)
    want = []
    for c in choices:
        starts = ops.expert_order(c, experts)[0]
        torch.cuda.synchronize()
        want.append(ops.grouped_linear_f8(rows8, w, starts))
        torch.cuda.synchronize()
    got = [ops.grouped_linear_f8(x, w, ops.expert_order(c, experts)[0]) for c in choices * 3]
    held = choices[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.grouped_linear_f8(x, w, ops.expert_order(held, experts)[0])
    for c in choices:
        held.copy_(c)
        graph.replay()
        got.append(y.clone())
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % len(want)]), i


@pytest.mark.gpu
def test_the_c_calls_over_bf16_rows(built_lib):
    from tinygpt_b200._lib import lib
    m, n, k = 5, 72, 264
    x, w, w3, bias = randn(m, k, seed=1), weight(n, k, seed=2), weight(n, k, 3, seed=3), randn(n, seed=4)
    starts = torch.tensor([0, 2, 2, 4], device="cuda", dtype=I32)
    rows = ops.f8_rows(x)
    q, scale, y = torch.empty_like(rows.q), torch.empty_like(rows.scale), torch.empty(m, n, device="cuda", dtype=BF16)
    (d, _), (d3, _) = ops._f8_desc(w, "test", 2), ops._f8_desc(w3, "test", 3)
    at = [t.data_ptr() for t in (y, q, scale, x)]
    assert lib().b200_f8_linear_of_bf16(*at, C.byref(d), bias.data_ptr(), m, _stream()) == 0
    assert torch.equal(y, ops.linear_f8(rows, w, bias)) and torch.equal(q.view(torch.uint8), rows.q.view(torch.uint8)) and torch.equal(scale, rows.scale)
    assert lib().b200_f8_grouped_of_bf16(*at, C.byref(d3), starts.data_ptr(), m, _stream()) == 0
    assert torch.equal(y, ops.grouped_linear_f8(rows, w3, starts))
    # refused, and nothing launched: a missing pointer, no rows, rows off the 16-byte boundary, a weight of the other kind
    y.fill_(7)
    for i in range(4):
        bad = [None if j == i else p for j, p in enumerate(at)]
        assert lib().b200_f8_linear_of_bf16(*bad, C.byref(d), None, m, _stream()) != 0
        assert lib().b200_f8_grouped_of_bf16(*bad, C.byref(d3), starts.data_ptr(), m, _stream()) != 0
    for bad, desc, rows_of in ((at, d, 0), (at, d, -1), ([at[0], at[1] + 8, *at[2:]], d, m), (at, d3, m)):
        assert lib().b200_f8_linear_of_bf16(*bad, C.byref(desc), None, rows_of, _stream()) != 0
    assert lib().b200_f8_grouped_of_bf16(*at, C.byref(d3), None, m, _stream()) != 0
    torch.cuda.synchronize()
    assert bool((y == 7).all())


def test_a_weight_too_large_for_fp32_is_refused():
    with pytest.raises(B200Error):
        ops.f8_quantize(torch.full((4, 4), 1e300, dtype=torch.float64))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 1152, 896), (48, 4096, 1440), (100, 520, 304)], ids=lambda v: str(v))
def test_given_rows_and_a_weight_written_in_front(built_lib, m, n, k):
    """Rows that are given: the first blocks of W are asked into L2 while the kernel in front, which may write W, still runs."""
    from tinygpt_b200._lib import check, lib
    raw, rows = [randn(n, k, seed=20 + i) for i in range(6)], [ops.f8_rows(randn(m, k, seed=50 + i)) for i in range(6)]
    now = ops.F8Weight(torch.empty(n, k, device="cuda", dtype=torch.uint8).view(rows[0].q.dtype), weight(n, k, seed=1).scale, n, k)
    junk = torch.empty(-(-k // 128), n, device="cuda")
    want = []
    for r, x in zip(raw, rows):
        w = now._replace(q=ops.f8_rows(r).q)
        torch.cuda.synchronize()
        want.append(ops.linear_f8(x, w))
        torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for r, x in zip(raw, rows):
            check(lib().b200_f8_rows_bf16(now.q.data_ptr(), junk.data_ptr(), r.data_ptr(), k, n, None, n, k, _stream()))
            got.append(ops.linear_f8(x, now))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % len(want)]), i
