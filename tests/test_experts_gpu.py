"""Routed experts (csrc/experts.cu): the order of the pairs, the sum back, and a whole layer in 8 bits — against their definitions."""
import pytest
import torch

import f8_oracle as orc
from test_f8_gpu import BF16, I32, gen, randn, weight
from tinygpt_b200 import ops
from tinygpt_b200._lib import B200Error


def choices(rows, top, experts, seed=0, missing=0.0):
    g = gen(seed)
    scores = torch.rand(rows, experts, generator=g, device="cuda") + 0.5 * torch.rand(experts, generator=g, device="cuda")
    chosen = scores.topk(top, 1).indices.to(I32)
    if missing:
        chosen[torch.rand(rows, top, generator=g, device="cuda") < missing] = -1
    return chosen.contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,top,experts", [(1, 1, 1), (1, 4, 32), (8, 2, 5), (33, 3, 7), (500, 4, 64), (300, 8, 1024), (4099, 2, 16), (20000, 8, 128)])
def test_order(built_lib, rows, top, experts):
    for missing in (0.0, 0.3):
        chosen = choices(rows, top, experts, rows, missing)
        starts, source, place = ops.expert_order(chosen, experts)
        flat = chosen.flatten().long()
        valid = flat >= 0
        order = torch.argsort(torch.where(valid, flat, torch.full_like(flat, experts)), stable=True)
        counts = torch.bincount(flat[valid], minlength=experts)
        n = int(counts.sum())
        assert starts.tolist() == [0] + counts.cumsum(0).tolist()
        assert torch.equal(source[:n].long(), order[:n] // top) and bool((source[n:] == -1).all())
        want = torch.full_like(flat, -1)
        want[order[:n]] = torch.arange(n, device="cuda")
        assert torch.equal(place.flatten().long(), want)


@pytest.mark.gpu
def test_order_of_odd_choices(built_lib):
    """One expert twice in a row, numbers past the experts, nothing chosen at all; no rows."""
    chosen = torch.tensor([[2, 2], [0, 2], [5, -7], [3, 1], [2 ** 31 - 1, -2 ** 31]], device="cuda", dtype=I32)
    got = [t.flatten().tolist() for t in ops.expert_order(chosen, 4)]
    assert got == [list(v) for v in orc.order(chosen.cpu(), 4)]
    starts, source, place = ops.expert_order(torch.full((7, 2), -1, device="cuda", dtype=I32), 3)
    assert not bool(starts.any()) and bool((source == -1).all()) and bool((place == -1).all())
    starts, source, place = ops.expert_order(chosen[:0], 4)
    assert starts.tolist() == [0] * 5 and source.shape == (0,) and place.shape == (0, 2)
    for bad in (lambda: ops.expert_order(chosen.long(), 4), lambda: ops.expert_order(chosen[0], 4), lambda: ops.expert_order(chosen, 1), lambda: ops.expert_order(chosen, 1025),
                lambda: ops.expert_order(chosen[:, :0], 4), lambda: ops.expert_order(chosen.cpu(), 4)):
        with pytest.raises(B200Error):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 8, 100, 200, 2056])
@pytest.mark.parametrize("rows,top", [(1, 1), (5, 4), (300, 2), (40, 9)])
def test_combine(built_lib, rows, top, n):
    y, g = randn(rows * top, n, seed=n), gen(rows)
    place = torch.randperm(rows * top, generator=g, device="cuda").to(I32).view(rows, top)
    place[0, 0] = -1
    place[-1, -1] = rows * top
    w = torch.rand(rows, top, generator=g, device="cuda")
    got = ops.expert_combine(y, place, w)
    valid = (place >= 0) & (place < rows * top)
    terms = y.double()[place.clamp(0, rows * top - 1).long()] * (w.double() * valid)[..., None]
    want, size = terms.sum(1), terms.abs().sum(1)
    assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + size * top * 2.0 ** -23 + 1e-38).all())
    y[int(place.flatten()[-1]) - 1, 0] = float("nan")
    for bad in (lambda: ops.expert_combine(y, place, w.double()), lambda: ops.expert_combine(y[1:], place, w), lambda: ops.expert_combine(y, place, w[:, :0]),
                lambda: ops.expert_combine(y.float(), place, w)):
        with pytest.raises(B200Error):
            bad()


def chain(x, chosen, weights, w_in, w_out):
    starts, source, place = ops.expert_order(chosen, w_in.q.shape[0])
    gu = ops.grouped_linear_f8(ops.f8_rows(x, source), w_in, starts)
    return ops.expert_combine(ops.grouped_linear_f8(ops.silu_mul_f8(gu), w_out, starts), place, weights)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,top,experts,width,ff", [(1, 1, 1, 8, 8), (1, 4, 32, 256, 128), (3, 2, 6, 100, 60), (8, 4, 32, 520, 264), (70, 3, 8, 200, 130), (300, 2, 16, 384, 256),
                                                       (1000, 4, 5, 260, 100)])
def test_layer(built_lib, rows, top, experts, width, ff):
    x, g = randn(rows, width, seed=rows), gen(ff)
    w_in, w_out = weight(2 * ff, width, experts, seed=1), weight(width, ff, experts, seed=2)
    for missing in (0.0, 0.4):
        chosen, weights = choices(rows, top, experts, rows, missing), torch.rand(rows, top, generator=g, device="cuda")
        got = ops.experts_f8(x, chosen, weights, w_in, w_out)
        assert torch.equal(got, chain(x, chosen, weights, w_in, w_out))
        # every pair by itself from the 8 bits of its row; [gate | up] and silu·up as the calls round them
        full_in, full_out, x8 = orc.dense(w_in), orc.dense(w_out), orc.held(ops.f8_rows(x))
        want, size = torch.zeros(rows, width, device="cuda", dtype=torch.float64), torch.zeros(rows, width, device="cuda", dtype=torch.float64)
        for e in range(experts):
            row, t = (chosen == e).nonzero(as_tuple=True)
            if not len(row):
                continue
            gu = x8[row] @ full_in[e].t()
            gate, up = gu[:, :ff], gu[:, ff:]
            a, w = gate / (1 + torch.exp(-gate)) * up, weights[row, t].double()[:, None]
            # how far a may be off: 2^-8 of gate and of up for their roundings to bf16 (silu's slope is at most 1.1), half a step of e4m3 (2^-4, and 2^-10 of the block's scale)
            off = a.abs() * 2.0 ** -4 * 1.01 + 1.1 * (2.0 ** -8 + 2.0 ** -13) * (gate.abs() * up.abs() + a.abs()) * 1.07 + orc.spread(orc.scales(a), ff) * 2.0 ** -10 * 1.1
            want.index_add_(0, row, w * (a @ full_out[e].t()))
            size.index_add_(0, row, w.abs() * (off @ full_out[e].abs().t() + (a @ full_out[e].t()).abs() * 2.0 ** -8))
        assert bool(((got.double() - want).abs() <= size * 1.01 + want.abs() * 2.0 ** -8 + 1e-30).all())
    none = ops.experts_f8(x, torch.full_like(chosen, -1), weights, w_in, w_out)
    assert not bool(none.any())
    assert ops.experts_f8(x[:0], chosen[:0], weights[:0], w_in, w_out).shape == (0, width)


@pytest.mark.gpu
def test_layer_refusals_and_captures(built_lib):
    x, w_in, w_out = randn(6, 136), weight(160, 136, 4, seed=1), weight(136, 80, 4, seed=2)
    chosen, weights = choices(6, 2, 4), torch.rand(6, 2, generator=gen(1), device="cuda")
    for bad in (lambda: ops.experts_f8(x, chosen, weights, w_out, w_in), lambda: ops.experts_f8(x[:5], chosen, weights, w_in, w_out),
                lambda: ops.experts_f8(x, chosen.long(), weights, w_in, w_out), lambda: ops.experts_f8(x, chosen, weights[:, :1], w_in, w_out),
                lambda: ops.experts_f8(x, chosen, weights, w_in, weight(136, 80, 3)), lambda: ops.experts_f8(x, chosen, weights, weight(160, 136), w_out),
                lambda: ops.experts_f8(x.float(), chosen, weights, w_in, w_out)):
        with pytest.raises(B200Error):
            bad()
    # two captured layers that may share torch's memory, replayed in turn
    pool = None
    graphs = []
    other = choices(6, 2, 4, seed=9)
    for c in (chosen, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = ops.experts_f8(x, c, weights, w_in, w_out)
        pool = graph.pool()
        graphs.append((graph, out, c))
    for _ in range(2):
        for graph, out, c in graphs:
            graph.replay()
            got = out.clone()
            assert torch.equal(got, ops.experts_f8(x, c, weights, w_in, w_out))
    # a NaN row spoils no other
    x2 = x.clone()
    x2[3, 4] = float("nan")
    got = ops.experts_f8(x2, chosen, weights, w_in, w_out)
    keep = torch.tensor([0, 1, 2, 4, 5], device="cuda")
    assert bool(got[3].isnan().all()) and torch.equal(got[keep], ops.experts_f8(x, chosen, weights, w_in, w_out)[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,top,experts,width,ff", [(700, 2, 4, 264, 256), (3000, 1, 3, 520, 128), (1500, 4, 32, 1000, 640), (2048, 4, 32, 512, 1024), (900, 2, 2, 136, 200)],
                         ids=lambda v: str(v))
def test_many_rows_are_the_steps(built_lib, rows, top, experts, width, ff):
    """Layers over many rows: the bits of the calls one behind the other, with choices that are none, an expert without rows, and rows that are not finite."""
    w_in, w_out = weight(2 * ff, width, experts, seed=1), weight(width, ff, experts, seed=2)
    x = randn(rows, width, seed=3)
    x[5, 7], x[rows - 1, 0], x[17] = float("inf"), float("nan"), 0.0
    chosen = torch.randint(-1, experts, (rows, top), generator=gen(4), device="cuda", dtype=I32)
    chosen[chosen == experts - 2] = experts - 1
    weights = torch.rand(rows, top, generator=gen(5), device="cuda")
    starts, source, place = ops.expert_order(chosen, experts)
    a = ops.silu_mul_f8(ops.grouped_linear_f8(ops.f8_rows(x, source), w_in, starts))
    want = ops.expert_combine(ops.grouped_linear_f8(a, w_out, starts), place, weights)
    for _ in range(2):
        got = ops.experts_f8(x, chosen, weights, w_in, w_out)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    fine = got[6 : rows - 1]
    assert bool(torch.isfinite(fine).all()) and bool((got[5].isnan() | (chosen[5] < 0).all()).all())
