"""Operators of 8 bits and of experts where they could go wrong: memory around what they write, offsets past 32 bits, very many experts, tiles of every kind with a bias and an
odd number of channels, two streams at once, which calls are native."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

import f8_oracle as orc
from test_f8_gpu import BF16, I32, each_group, gen, groups, randn, weight
from tinygpt_b200 import ops

ROOT = Path(__file__).resolve().parent.parent


def test_the_weight_s_descriptor_is_the_compiler_s(tmp_path):
    from tinygpt_b200 import _lib
    src, exe = tmp_path / "sz.c", tmp_path / "sz"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b200_decode.h"\nint main(void) { printf("%zu %zu %zu", sizeof(b200_f8_weight), '
                   "offsetof(b200_f8_weight, n), offsetof(b200_f8_weight, experts)); return 0; }\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == [C.sizeof(_lib.F8Desc), _lib.F8Desc.n.offset, _lib.F8Desc.experts.offset]


@pytest.mark.gpu
def test_plain_calls_are_native(built_lib):
    x, w, w3 = randn(6, 256), weight(64, 256), weight(64, 256, 2)
    rows, starts = ops.f8_rows(x), torch.tensor([0, 2, 6], device="cuda", dtype=I32)
    f = ops._fast
    assert f.f8_rows(x).__class__ is tuple and f.norm_f8(x, x, None, 1e-6).__class__ is tuple and f.silu_mul_f8(x).__class__ is tuple
    assert torch.equal(f.f8_rows_dequantize(*rows), ops.f8_rows_dequantize(rows))
    for got in (f.linear_f8(*rows, *w, None), f.linear_f8(x, None, None, *w, None)):
        assert torch.equal(got, ops.linear_f8(rows, w))
    assert torch.equal(f.grouped_linear_f8(*rows, *w3, starts), ops.grouped_linear_f8(x, w3, starts))
    assert f.grouped_linear(x, randn(2, 8, 256), starts).shape == (6, 8)
    # what is not plain goes the other way, with the same result
    assert f.f8_rows(x.t()) is None and f.linear_f8(x.t(), None, None, *w, None) is None
    wide = randn(6, 512)
    assert torch.equal(ops.linear_f8(wide[:, :256], w), ops.linear_f8(wide[:, :256].contiguous(), w))
    assert torch.equal(ops.linear_f8(rows, w._replace(q=w.q.t().contiguous().t())), ops.linear_f8(rows, w))


SHAPES = [(1, 130, 300), (5, 64, 2000), (40, 257, 520), (100, 1000, 260), (130, 72, 1100), (260, 2051, 130), (3000, 517, 260)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SHAPES, ids=lambda v: str(v))
def test_linear_writes_its_rows_alone(built_lib, m, n, k):
    from tinygpt_b200._lib import check, lib
    w, x, bias = weight(n, k, seed=1), ops.f8_rows(randn(m, k, seed=2)), randn(n, seed=3)
    d, _ = ops._f8_desc(w, "test", 2)
    want = ops.linear_f8(x, w, bias)
    orc.close(want, orc.held(x), orc.dense(w), bias)
    for off in (64, 65, 68, 72):   # results at other addresses than torch's
        box = torch.full((m * n + 256,), 7.0, device="cuda", dtype=BF16)
        check(lib().b200_f8_linear_bf16(box[off:].data_ptr(), x.q.data_ptr(), x.scale.data_ptr(), C.byref(d), bias.data_ptr(), m, torch.cuda.current_stream().cuda_stream))
        assert bool((box[:off] == 7).all()) and bool((box[off + m * n :] == 7).all()) and torch.equal(box[off : off + m * n].view(m, n), want)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [(0, 1, 30, 17), (100, 0, 3, 60), (300, 129, 0, 1000), (5000, 1, 3000, 0)], ids=str)
@pytest.mark.parametrize("n,k", [(72, 136), (1000, 264), (2053, 128)])
def test_groups_write_their_rows_alone(built_lib, counts, n, k):
    from tinygpt_b200._lib import check, lib
    starts, rows = groups(counts, 2, 5)
    x, w8 = randn(rows, k), weight(n, k, 4, seed=1)
    x8, w = ops.f8_rows(x), (torch.randn(4, n, k, generator=gen(2), device="cuda") / 8).to(BF16)
    d, _ = ops._f8_desc(w8, "test", 3)
    st = torch.cuda.current_stream().cuda_stream
    for call, xs, ws in ((lambda y: lib().b200_f8_grouped_bf16(y, x8.q.data_ptr(), x8.scale.data_ptr(), C.byref(d), starts.data_ptr(), rows, st), orc.held(x8), orc.dense(w8)),
                         (lambda y: lib().b200_grouped_bf16(y, x.data_ptr(), w.data_ptr(), starts.data_ptr(), rows, 4, n, k, st), x.double(), w.double())):
        box = torch.full((rows * n + 128,), 7.0, device="cuda", dtype=BF16)
        check(call(box[64:].data_ptr()))
        assert bool((box[:64] == 7).all()) and bool((box[64 + rows * n :] == 7).all())
        each_group(box[64 : 64 + rows * n].view(rows, n), xs, ws, starts)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3000, 5001, 300), (2500, 4099, 129), (2000, 6000, 1000)])
def test_many_rows_with_a_bias(built_lib, m, n, k):
    w, x, bias = weight(n, k, seed=1), ops.f8_rows(randn(m, k, seed=2)), randn(n, seed=3)
    orc.close(ops.linear_f8(x, w, bias), orc.held(x), orc.dense(w), bias)


@pytest.mark.gpu
@pytest.mark.parametrize("experts,each", [(513, 40), (600, 150), (1024, 3), (1024, 0)])
def test_very_many_experts(built_lib, experts, each):
    """Up to 1 024 matrices, where the tables of the groups are largest; the ways for few and for many matrices meet at 512."""
    n, k = 136, 128
    counts = [(each * (e % 3) + (e == 7)) for e in range(experts)]
    starts, rows = groups(counts, 0, 3)
    x, w8 = randn(rows, k, seed=each), weight(n, k, experts, seed=1)
    w = (torch.randn(experts, n, k, generator=gen(2), device="cuda") / 8).to(BF16)
    x8 = ops.f8_rows(x)
    owner = torch.repeat_interleave(torch.arange(experts, device="cuda"), torch.tensor(counts, device="cuda"))
    for y, xs, ws in ((ops.grouped_linear_f8(x8, w8, starts), orc.held(x8), orc.dense(w8)), (ops.grouped_linear(x, w, starts), x.double(), w.double())):
        assert not bool(y[rows - 3 :].any())
        for first in range(0, rows - 3, 4096):
            rest = slice(first, min(first + 4096, rows - 3))
            xe, we = xs[rest], ws[owner[rest]]
            want, size = torch.einsum("rk,rnk->rn", xe, we), torch.einsum("rk,rnk->rn", xe.abs(), we.abs())
            # half a step of bf16 and the fp32 sums', as f8_oracle.close has them
            assert bool(((y[rest].double() - want).abs() <= want.abs() * 2.0 ** -8 + size * ((k + 32) * 2.0 ** -23) + 1e-38).all())


@pytest.mark.gpu
def test_offsets_past_32_bits(built_lib):
    """Results and rows of more than 2^31 entries: the last ones are those of a small call."""
    rows, n = 140_000, 16_384
    w = weight(n, 16)
    x = randn(rows, 16)
    y = ops.linear_f8(x, w)
    assert y.numel() > 2 ** 31
    for first in (0, 131_000, rows - 200):
        orc.close(y[first : first + 200], orc.held(ops.f8_rows(x[first : first + 200])), orc.dense(w))
    got, (norm, z), silu = ops.f8_rows(y), ops.add_rms_norm_f8(y, y, None, 1e-6), ops.silu_mul_f8(y)
    last = y[-3:].clone()
    small, (small_norm, small_z), small_silu = ops.f8_rows(last), ops.add_rms_norm_f8(last, last, None, 1e-6), ops.silu_mul_f8(last)
    for a, b in ((got, small), (norm, small_norm), (silu, small_silu)):
        assert torch.equal(a.q[-3:].view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.scale[:, -3:], b.scale)
    assert torch.equal(z[-3:], small_z)
    del norm, z, silu
    back = ops.f8_rows_dequantize(got)
    assert torch.equal(back[-3:], ops.f8_rows_dequantize(small))
    place = torch.arange(rows, device="cuda", dtype=I32).view(-1, 2).flip(1).contiguous()
    out = ops.expert_combine(y, place, torch.ones(rows // 2, 2, device="cuda"))
    assert torch.equal(out[-1], (y[-1].float() + y[-2].float()).to(BF16))


@pytest.mark.gpu
def test_two_streams_at_once(built_lib):
    """Calls of two streams that meet on the SMs, clusters among them: every one gives what it gives alone."""
    w = [weight(1000, 4096, seed=i) for i in range(2)]
    w3 = [weight(264, 520, 6, seed=i) for i in range(2)]
    xs = [[randn(m, 4096, seed=m + i) for m in (1, 40, 130, 700)] for i in range(2)]
    starts = torch.tensor([0, 3, 3, 50, 51, 300, 310], device="cuda", dtype=I32)
    xg = [randn(310, 520, seed=7 + i) for i in range(2)]

    def calls(i):
        return [ops.linear_f8(x, w[i]) for x in xs[i]] + [ops.grouped_linear_f8(xg[i], w3[i], starts), ops.f8_rows_dequantize(ops.rms_norm_f8(xg[i], None, 1e-6))]

    want = [calls(0), calls(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(calls(i))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


@pytest.mark.gpu
def test_an_expert_twice_in_a_row_and_a_padded_batch(built_lib):
    width, ff, experts = 264, 136, 5
    w_in, w_out = weight(2 * ff, width, experts, seed=1), weight(width, ff, experts, seed=2)
    x = randn(7, width)
    chosen = torch.tensor([[2, 2], [0, 1], [4, 4], [-1, 3], [-1, -1], [3, 9], [1, 0]], device="cuda", dtype=I32)
    weights = torch.rand(7, 2, generator=gen(3), device="cuda")
    got = ops.experts_f8(x, chosen, weights, w_in, w_out)
    one = ops.experts_f8(x, chosen[:, :1].contiguous(), torch.ones(7, 1, device="cuda"), w_in, w_out).double()
    # the same expert twice: the sum of its weights; both terms and the sum in fp32, the expert's row rounded to bf16 once
    for r in (0, 2):
        want = one[r] * weights[r].double().sum()
        assert bool(((got[r].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -22) + 1e-38).all())
    assert not bool(got[4].any())
    # a padded batch may be cut in another way, whose sums differ in fp32: steps of bf16 in gate and up (2^-8 each) and, where those cross one, of e4m3 in single entries of a
    # block (2^-3 of one of 136 terms of random signs)
    padded = ops.experts_f8(torch.cat([x, x]), torch.cat([chosen, torch.full_like(chosen, -1)]), torch.cat([weights, weights]), w_in, w_out)
    assert not bool(padded[7:].any())
    assert bool(((padded[:7].double() - got.double()).abs() <= 2.0 ** -6 * got.double().abs().amax(1, keepdim=True)).all())
