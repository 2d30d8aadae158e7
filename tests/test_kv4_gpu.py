"""The paged cache of 4-bit keys and values (csrc/kv4*.cu) against tests/kv4_oracle.py: what is stored bit by bit, the attention over it at head sizes, groups,
lengths, masks and batches where it can go wrong, the bookkeeping of pages against lists, and all of them together as a server uses them."""
import random

import pytest
import torch

import kv4_oracle as orc
from tinygpt_b200 import ops
from tinygpt_b200._lib import B200Error

BF16 = torch.bfloat16


def dev(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def starts_of(counts):
    s = [0]
    for c in counts:
        s.append(s[-1] + c)
    return dev(s)


class Rand:
    def __init__(self, seed=0):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def __call__(self, *shape, spread=1.0, mean=0.0):
        return (torch.randn(*shape, generator=self.g, device="cuda") * spread + mean).to(BF16)


def filled(rand, lengths, kv_heads, dim, layers=1, layer=0, spare=2, seqs=None, room=1):
    """A cache whose sequences came in two steps, so that their pages lie mixed; k and v as given."""
    n = len(lengths)
    pages = sum(-(-l // 64) for l in lengths) + spare
    cache = ops.kv4_cache(layers, pages, n, max(max(-(-l // 64) for l in lengths), 1) + room, kv_heads, dim)
    cache.pages.fill_(255)   # values 15, scale and middle NaN: what is not written must not be seen
    k, v = rand(sum(lengths), kv_heads, dim, spread=1.5, mean=0.7), rand(sum(lengths), kv_heads, dim)
    order = dev(list(range(n)) if seqs is None else seqs)
    half = [l // 3 for l in lengths]
    assert ops.kv4_extend(cache, order, dev(half)).tolist() == [0] * n
    assert ops.kv4_extend(cache, order, dev([l - h for l, h in zip(lengths, half)])).tolist() == half
    ops.kv4_store(cache, layer, k, v, order, starts_of(lengths), dev([0] * n))
    return cache, order, k, v


def run_case(rand, lengths, counts, heads, kv_heads, dim, window=0, scale=None, layers=1, layer=0, room=1):
    cache, seqs, k, v = filled(rand, lengths, kv_heads, dim, layers, layer, room=room)
    q = rand(max(sum(counts), 1), heads, dim)
    pos = [l - c if l else -1 for l, c in zip(lengths, counts)]
    out = ops.kv4_attention(cache, layer, q, seqs, starts_of(counts), dev(pos), window=window, scale=scale)
    hk, hv = orc.held(k), orc.held(v)
    row = first = 0
    for length, count, p in zip(lengths, counts, pos):
        want, bound = orc.attention(q[row:row + count], hk[first:first + length], hv[first:first + length], p, scale or dim ** -0.5, window)
        err = (out[row:row + count].cpu().double() - want).abs()
        assert bool((err <= bound).all()), (length, count, float((err / bound.clamp(min=1e-30)).max()))
        row, first = row + count, first + length
    assert not out[row:].any()
    return cache, q, seqs, pos, out


# ------------------------------------------------------------------------------------------------- without a device
def test_refusals_without_a_device():
    with pytest.raises(B200Error, match="heads of 80"):
        ops.kv4_cache(1, 4, 2, 2, 2, 80)
    with pytest.raises(B200Error, match="n_pages"):
        ops.kv4_cache(1, 0, 2, 2, 2, 64)
    for call in (lambda: ops.kv4_free(None, None), lambda: ops.kv4_extend(3, None, None), lambda: ops.kv4_compact(None),
                 lambda: ops.kv4_store(None, 0, None, None, None, None, None), lambda: ops.kv4_attention(None, 0, None, None, None, None)):
        with pytest.raises(B200Error, match="KV4Cache"):
            call()
    if not torch.cuda.is_available():
        with pytest.raises(B200Error):
            ops.kv4_cache(1, 4, 2, 2, 2, 64)


def test_descriptors_match_the_compiler(tmp_path):
    import ctypes as C
    import subprocess
    from pathlib import Path
    from tinygpt_b200._lib import KV4Desc, W4Desc
    (tmp_path / "sz.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b200_decode.h"\nint main(void) { printf("%zu %zu %zu %zu %zu %zu\\n", '
                                   'sizeof(b200_w4_weight), offsetof(b200_w4_weight, group), sizeof(b200_kv4_cache), offsetof(b200_kv4_cache, refs), '
                                   'offsetof(b200_kv4_cache, layers), offsetof(b200_kv4_cache, dim)); return 0; }\n')
    subprocess.run(["gcc", "-I", str(Path(__file__).resolve().parent.parent / "include"), str(tmp_path / "sz.c"), "-o", str(tmp_path / "sz")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "sz")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(W4Desc), W4Desc.group.offset, C.sizeof(KV4Desc), KV4Desc.refs.offset, KV4Desc.layers.offset, KV4Desc.dim.offset]


def test_page_bytes(built_lib):
    from tinygpt_b200._lib import lib
    assert [lib().b200_kv4_page_bytes(8, d) for d in (64, 128, 192, 256)] == [2 * 8 * 64 * (d // 2 + d // 64 * 4) for d in (64, 128, 192, 256)]
    assert lib().b200_kv4_page_bytes(1, 32) == -1 and lib().b200_kv4_page_bytes(0, 64) == -1


# ------------------------------------------------------------------------------------------------- rows in and out
@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads,dim", [(1, 64), (3, 128), (2, 192), (2, 256)])
def test_store_and_load(built_lib, kv_heads, dim):
    rand = Rand(1)
    firsts, counts = [0, 5, 63, 64, 100, 0], [1, 60, 2, 130, 0, 77]
    n = len(firsts)
    cache = ops.kv4_cache(2, 32, 8, 6, kv_heads, dim)
    seqs = dev([6, 1, 0, 3, 7, 2])
    ops.kv4_extend(cache, seqs, dev(firsts))
    pos = ops.kv4_extend(cache, seqs, dev(counts))
    assert pos.tolist() == firsts
    cache.pages.zero_()
    before = cache.pages[0].clone()
    rows = sum(counts) + 3   # three rows of nobody
    wide = rand(rows, 3 * kv_heads * dim, spread=2.0)
    k, v = (wide[:, i * kv_heads * dim:(i + 1) * kv_heads * dim].unflatten(1, (kv_heads, dim)) for i in (0, 2))
    k[0, 0, :64] = 3.0             # a group of one number
    k[2, 0, 5], v[4, 0, 7] = float("inf"), float("nan")
    v[6, 0, :64] = torch.linspace(-3e38, 3e38, 64, device="cuda").to(BF16)
    v[7, 0, :64] = torch.linspace(1e-40, 9e-40, 64, device="cuda").to(BF16)
    ops.kv4_store(cache, 1, k, v, seqs, starts_of(counts), pos)
    assert torch.equal(cache.pages[0], before)   # the other layer
    for got, x in zip(ops.kv4_load(cache, 1, seqs, starts_of(counts), pos, rows), (k, v)):
        want = orc.held(x)
        want[sum(counts):] = 0
        got = got.cpu()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
        plain = x.cpu().float()[8:sum(counts)]
        span = plain.unflatten(-1, (-1, 64))
        span = (span.amax(-1) - span.amin(-1)).repeat_interleave(64, -1)
        # half a step, and what the roundings of scale (15 steps of it) and middle (of size lo + 8·scale) move
        assert bool(((got[8:sum(counts)] - plain).abs() <= span / 15 * (0.5 + 15 * 2.0 ** -8) + plain.abs().amax() * 2.0 ** -8).all())


@pytest.mark.gpu
def test_rows_without_a_place(built_lib):
    rand = Rand(2)
    cache = ops.kv4_cache(1, 6, 3, 3, 2, 64)
    seqs = dev([0, 1, 2])
    assert ops.kv4_extend(cache, seqs, dev([70, 10, 0])).tolist() == [0, 0, 0]
    k, v = rand(12, 2, 64), rand(12, 2, 64)
    cache.pages.zero_()
    # sequence 0 past its pages at 128 …, sequence 1 refused, a number outside, a place past the table
    for s, p in (([0, 1, 2], [126, -1, 0]), ([7, -3, 0], [0, 0, 192]), ([0, 1, 2], [2 ** 31 - 1, 64, 2 ** 30])):
        ops.kv4_store(cache, 0, k, v, dev(s), dev([0, 4, 8, 12]), dev(p))
        got = ops.kv4_load(cache, 0, dev(s), dev([0, 4, 8, 12]), dev(p), 12)[0].cpu()
        if p[0] == 126:
            assert torch.equal(got[:2], orc.held(k[:2]))
            got[:2] = 0
        assert not got.any()
    # a shared page takes no rows
    assert ops.kv4_fork(cache, dev([0]), dev([2])).tolist() == [1]
    was = cache.pages.clone()
    ops.kv4_store(cache, 0, k[:4], v[:4], dev([2]), dev([0, 4]), dev([60]))
    first = cache.table[0, 0]
    assert torch.equal(was[0, first], cache.pages[0, first])
    ops.kv4_store(cache, 0, k[:4], v[:4], dev([2]), dev([0, 4]), dev([64]))
    assert torch.equal(ops.kv4_load(cache, 0, dev([2]), dev([0, 4]), dev([64]), 4)[0].cpu(), orc.held(k[:4]))


# ------------------------------------------------------------------------------------------------- attention
# room: pages that a sequence could still take.  Calls over small caches go to clusters, others are cut evenly over the GPU's warps.
@pytest.mark.gpu
@pytest.mark.parametrize("room", [1, 9000])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (14, 2, 64), (4, 2, 128), (16, 2, 128), (9, 1, 128), (6, 2, 192), (10, 1, 192), (8, 4, 256), (20, 2, 256)])
def test_single_tokens(built_lib, heads, kv_heads, dim, room):
    lengths = [1, 15, 16, 17, 0, 63, 64, 65, 130, 511, 700]
    run_case(Rand(3), lengths, [1] * len(lengths), heads, kv_heads, dim, room=room)


@pytest.mark.gpu
@pytest.mark.parametrize("n,heads,kv_heads,dim", [(1, 4, 1, 64), (8, 4, 2, 128), (9, 8, 4, 64), (35, 3, 1, 128), (18, 32, 4, 64), (74, 2, 2, 64), (2, 24, 2, 256)])
def test_clusters_of_all_sizes(built_lib, n, heads, kv_heads, dim):
    """One to eight CTAs to a sequence's head, sequences of which most have fewer steps than the cluster has warps."""
    lengths = [(37 * i) % 400 + (i % 3 > 0) for i in range(n)]
    run_case(Rand(12), lengths, [1] * n, heads, kv_heads, dim, window=0 if n % 2 else 70)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [([4500], 8, 1, 64), ([9000, 1, 4097], 6, 2, 128), ([8200], 12, 6, 64), ([4200, 4099], 16, 2, 192)])
def test_clusters_of_sixteen(built_lib, lengths, heads, kv_heads, dim):
    """Few heads over long caches: 128 warps to a sequence's head, of which a short neighbour needs one."""
    run_case(Rand(14), lengths, [1] * len(lengths), heads, kv_heads, dim, window=0)


@pytest.mark.gpu
@pytest.mark.parametrize("room", [1, 9000])
def test_unequal_counts_of_few_columns(built_lib, room):
    """Sequences that bring several blocks of columns where the average brings one; the last rows are nobody's."""
    run_case(Rand(13), [100, 300, 5, 64, 1], [3, 11, 0, 1, 0], 4, 2, 64, room=room)
    run_case(Rand(13), [100, 300, 5, 64, 90], [0, 50, 0, 1, 0], 2, 2, 128, room=room)


@pytest.mark.gpu
@pytest.mark.parametrize("room", [1, 9000])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (7, 1, 64), (8, 2, 128), (4, 2, 192), (4, 1, 256)])
@pytest.mark.parametrize("window", [0, 1, 40, 200])
def test_several_tokens(built_lib, heads, kv_heads, dim, window, room):
    run_case(Rand(4), [3, 64, 200, 90, 330], [3, 2, 70, 0, 33], heads, kv_heads, dim, window=window, room=room)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,counts,heads,kv_heads,dim", [([700], [700], 8, 1, 64), ([520, 900, 1], [520, 333, 1], 6, 2, 128), ([40 + i for i in range(40)], [40] * 40, 8, 2, 64),
                                                               ([300], [300], 4, 2, 256)])
@pytest.mark.parametrize("window", [0, 1, 90])
def test_prompts(built_lib, lengths, counts, heads, kv_heads, dim, window):
    """Rows from a sequence's first token on: blocks of columns that see from one step to all, more of them than a warp has lanes, empty ones under a window."""
    run_case(Rand(15), lengths, counts, heads, kv_heads, dim, window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[6000], [5000, 64, 2000], [700] * 40])
def test_work_cut_over_ctas(built_lib, lengths):
    rand = Rand(5)
    cache, q, seqs, pos, out = run_case(rand, lengths, [1] * len(lengths), 4, 2, 64, layers=2, layer=1, scale=0.05, room=9000)
    again = ops.kv4_attention(cache, 1, q, seqs, starts_of([1] * len(lengths)), dev(pos), scale=0.05)
    assert torch.equal(out, again)


@pytest.mark.gpu
def test_largest_scores_come_late_and_early(built_lib):
    """Running maxima that move with every page, weights that vanish against a later one, equal scores everywhere."""
    rand = Rand(6)
    for kind in ("up", "down", "equal", "low"):
        cache, seqs, k, v = filled(rand, [400], 1, 64)
        x = torch.linspace(-40, 40, 400, device="cuda")
        if kind == "down":
            x = x.flip(0)
        if kind == "equal":
            x = torch.zeros_like(x)
        if kind == "low":
            x = x * 0 - 3e4
        k = (x[:, None, None] * torch.ones(1, 1, 64, device="cuda")).to(BF16)
        ops.kv4_store(cache, 0, k, v, seqs, dev([0, 400]), dev([0]))
        q = torch.ones(1, 2, 64, device="cuda", dtype=BF16)
        out = ops.kv4_attention(cache, 0, q, seqs, dev([0, 1]), dev([399]))
        want, bound = orc.attention(q, orc.held(k), orc.held(v), 399, 0.125, 0)
        assert bool(((out.cpu().double() - want).abs() <= bound).all()), kind


@pytest.mark.gpu
def test_what_is_not_seen_does_not_count(built_lib):
    """NaN and infinities in pages behind the length, in positions behind a row's own and in front of its window; in what is seen they do count."""
    rand = Rand(7)
    heads, kv_heads, dim = 4, 2, 64
    cache, seqs, k, v = filled(rand, [200], kv_heads, dim)
    q = rand(3, heads, dim)
    args = (cache, 0, q, seqs, dev([0, 3]), dev([100]))
    bad = torch.full((1, kv_heads, dim), float("nan"), device="cuda", dtype=BF16)
    want, windowed = ops.kv4_attention(*args), ops.kv4_attention(*args, window=20)
    ops.kv4_store(cache, 0, bad, bad, seqs, dev([0, 1]), dev([103]))
    ops.kv4_store(cache, 0, bad * float("inf"), bad, seqs, dev([0, 1]), dev([80]))
    assert torch.equal(windowed, ops.kv4_attention(*args, window=20))
    ops.kv4_store(cache, 0, k[80:81], v[80:81], seqs, dev([0, 1]), dev([80]))
    assert torch.equal(want, ops.kv4_attention(*args))
    ops.kv4_store(cache, 0, bad, bad, seqs, dev([0, 1]), dev([102]))
    got = ops.kv4_attention(*args)
    assert torch.equal(got[:2], want[:2]) and bool(got[2].isnan().all())
    ops.kv4_store(cache, 0, bad.expand(200, -1, -1).contiguous(), v, seqs, dev([0, 200]), dev([0]))
    assert bool(ops.kv4_attention(*args).isnan().all())
    nan_q = q.clone()
    nan_q[1, 2] = float("nan")
    ops.kv4_store(cache, 0, k, v, seqs, dev([0, 200]), dev([0]))
    got, keep = ops.kv4_attention(cache, 0, nan_q, *args[3:]), torch.ones(3, heads, dtype=torch.bool)
    keep[1, 2] = False
    assert torch.equal(got.cpu()[keep], want.cpu()[keep]) and bool(got[1, 2].isnan().all())


@pytest.mark.gpu
def test_rows_that_see_nothing(built_lib):
    rand = Rand(8)
    cache, seqs, k, v = filled(rand, [70, 0, 5], 2, 64)
    q = rand(9, 4, 64)
    # rows in front of the first sequence and behind the last one; an empty sequence; a refused one; a number outside the cache
    out = ops.kv4_attention(cache, 0, q, dev([0, 1, 2, 9, -1]), dev([1, 3, 4, 5, 6, 7]), dev([68, 0, -1, 3, 3]))
    assert bool(out[1:3].any()) and not out[0].any() and not out[3:].any()
    # a table whose pages are bad numbers
    cache.table[0, 0] = cache.n_pages + 5
    cache.table[0, 1] = -7
    assert not ops.kv4_attention(cache, 0, q[:1], dev([0]), dev([0, 1]), dev([69])).any()
    # a window that ends before what the sequence holds
    assert not ops.kv4_attention(cache, 0, q[:1], dev([2]), dev([0, 1]), dev([500]), window=10).any()


@pytest.mark.gpu
@pytest.mark.parametrize("room", [1, 9000])
def test_strides_streams_capture_and_refusals(built_lib, room):
    rand = Rand(9)
    cache, seqs, k, v = filled(rand, [150, 40], 2, 128, room=room)
    wide = rand(2, 3 * 4 * 128)
    q = wide[:, 512:1024].unflatten(1, (4, 128))
    where = (seqs, dev([0, 1, 2]), dev([149, 39]))
    want = ops.kv4_attention(cache, 0, q.contiguous(), *where)
    assert torch.equal(ops.kv4_attention(cache, 0, q, *where), want)
    assert torch.equal(ops.kv4_attention(cache, 0, q.transpose(1, 2).contiguous().transpose(1, 2), *where), want)
    off = torch.empty(4 + q.numel(), device="cuda", dtype=BF16)[4:].view(q.shape)   # off the 16-byte boundary
    off.copy_(q)
    assert torch.equal(ops.kv4_attention(cache, 0, off, *where), want)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(st):
        x = q.contiguous()
        for _ in range(2):   # two graphs at once, over one cache
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                pos = ops.kv4_extend(cache, seqs, torch.ones_like(seqs))
                ops.kv4_store(cache, 0, x[:, :2], x[:, 2:], seqs, where[1], pos)
                outs.append(ops.kv4_attention(cache, 0, x, seqs, where[1], pos))
            graphs.append(graph)
        graphs[1].replay()
        graphs[0].replay()
    st.synchronize()
    assert cache.length.tolist() == [152, 42]
    hk, hv = (torch.cat((orc.held(t[:150]), orc.held(y.repeat(2, 1, 1)))) for t, y in ((k, x[:1, :2]), (v, x[:1, 2:])))
    for out, at in ((outs[1], 150), (outs[0], 151)):
        ref, bound = orc.attention(x[:1], hk[:at + 1], hv[:at + 1], at, 128 ** -0.5, 0)
        assert bool(((out[:1].cpu().double() - ref).abs() <= bound).all())
    for bad in (lambda: ops.kv4_attention(cache, 1, q, *where), lambda: ops.kv4_attention(cache, -1, q, *where), lambda: ops.kv4_attention(cache, 2 ** 70, q, *where),
                lambda: ops.kv4_attention(cache, 0, q.float(), *where), lambda: ops.kv4_attention(cache, 0, q[:, :3], *where),
                lambda: ops.kv4_attention(cache, 0, q[..., :64], *where), lambda: ops.kv4_attention(cache, 0, q, seqs.long(), *where[1:]),
                lambda: ops.kv4_attention(cache, 0, q, seqs, where[1][:2], where[2]), lambda: ops.kv4_attention(cache, 0, q, *where, window=-1),
                lambda: ops.kv4_attention(cache, 0, q, *where, scale=0.0), lambda: ops.kv4_attention(cache, 0, q, *where, scale=float("nan")),
                lambda: ops.kv4_store(cache, 0, q, q, *where), lambda: ops.kv4_store(cache, 0, q[:, :2], q[:1, :2], *where),
                lambda: ops.kv4_store(cache, 1, q[:, :2], q[:, :2], *where), lambda: ops.kv4_load(cache, 0, *where, -1),
                lambda: ops.kv4_extend(cache, seqs, dev([1])), lambda: ops.kv4_extend(cache, seqs.cpu(), dev([1, 1])), lambda: ops.kv4_free(cache, seqs.float()),
                lambda: ops.kv4_extend(cache, dev([0] * 1025), dev([0] * 1025)), lambda: setattr(cache, "table", cache.table.clone())):
        with pytest.raises((B200Error, AttributeError)):
            bad()
    none = dev([])
    assert ops.kv4_extend(cache, none, none).shape == (0,) and ops.kv4_free(cache, none) is None
    assert ops.kv4_attention(cache, 0, q[:0], *where).shape == (0, 4, 128) and ops.kv4_load(cache, 0, *where, 0)[0].shape == (0, 2, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("room", [1, 9000])
def test_places_past_32_bits(built_lib, room):
    """A pool of 7 GB: pages and layers whose places no 32 bits hold."""
    rand = Rand(14)
    cache = ops.kv4_cache(3, 16000, 3, 3 + room, 8, 256)
    assert cache.pages[0].numel() * 2 > 2 ** 32
    cache.table[:, :3] = dev([[15999, 3, 15000], [15998, -1, -1], [7, 15997, -1]])
    cache.length.copy_(dev([150, 20, 100]))
    cache.refs[dev([15999, 3, 15000, 15998, 7, 15997]).long()] = 1
    lengths, seqs = [150, 20, 100], dev([0, 1, 2])
    k, v, q = rand(270, 8, 256), rand(270, 8, 256), rand(3, 16, 256)
    ops.kv4_store(cache, 2, k, v, seqs, starts_of(lengths), dev([0, 0, 0]))
    assert torch.equal(ops.kv4_load(cache, 2, seqs, starts_of(lengths), dev([0, 0, 0]), 270)[1].cpu(), orc.held(v))
    out, first = ops.kv4_attention(cache, 2, q, seqs, dev([0, 1, 2, 3]), dev([l - 1 for l in lengths])), 0
    for i, l in enumerate(lengths):
        want, bound = orc.attention(q[i:i + 1], orc.held(k[first:first + l]), orc.held(v[first:first + l]), l - 1, 1 / 16, 0)
        assert bool(((out[i:i + 1].cpu().double() - want).abs() <= bound).all())
        first += l
    before = cache.pages[2, 15999].clone()
    assert ops.kv4_compact(cache).tolist() == [6]
    assert torch.equal(cache.pages[2, cache.table[0, 0]], before) and int(cache.table.max()) < 6
    assert torch.equal(ops.kv4_attention(cache, 2, q, seqs, dev([0, 1, 2, 3]), dev([l - 1 for l in lengths])), out)


@pytest.mark.gpu
def test_a_chain_beside_the_ends_of_kernels(built_lib):
    """Launches that begin while the one in front ends read what it wrote: a decode loop without a synchronisation against the same with one after every call."""
    def chain(sync, room):
        rand = Rand(15)
        s = (lambda t: (torch.cuda.synchronize(), t)[1]) if sync else (lambda t: t)
        hidden, heads, kv_heads, dim, n = 256, 4, 2, 64, 5
        w_in, w_out = ops.w4_quantize(rand((heads + 2 * kv_heads) * dim, hidden, spread=0.06)), ops.w4_quantize(rand(hidden, heads * dim, spread=0.06), group=128)
        cache, seqs, starts = ops.kv4_cache(1, 60, n + 1, 4 + room, kv_heads, dim), dev(list(range(n))), dev(list(range(n + 1)))
        cache.pages.zero_()
        x, out = rand(n, hidden), []
        for step in range(70):
            pos = s(ops.kv4_extend(cache, seqs, dev([1] * n)))
            q, k, v = (t.unflatten(1, (-1, dim)) for t in s(ops.linear_w4(x, w_in)).split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
            ops.kv4_store(cache, 0, k, v, seqs, starts, pos)
            x = s(ops.add(x, s(ops.linear_w4(s(ops.kv4_attention(cache, 0, q, seqs, starts, pos)).flatten(1), w_out))))
            x = s(ops.rms_norm(x, None, 1e-6))
            if step % 20 == 10:
                s(ops.kv4_fork(cache, dev([2]), dev([n])))
                ops.kv4_free(cache, dev([0]))
                s(ops.kv4_compact(cache))
                s(ops.kv4_fork(cache, dev([n]), dev([0])))
                ops.kv4_free(cache, dev([n]))
            out.append(x)
        return torch.stack(out), cache
    for room in (1, 9000):
        want, ref = chain(True, room)
        assert bool(torch.isfinite(want.float()).all())
        for _ in range(5):
            got, cache = chain(False, room)
            assert torch.equal(got, want) and torch.equal(cache.table, ref.table) and torch.equal(cache.refs, ref.refs) and torch.equal(cache.length, ref.length)


# ------------------------------------------------------------------------------------------------- pages
@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(8))
def test_bookkeeping_against_lists(built_lib, seed):
    rng = random.Random(seed)
    n_pages, n_seqs, max_pages = rng.choice([(40, 6, 9), (5000, 40, 300), (9000, 200, 64), (17, 3, 17), (4096, 60, 90)])
    cache, model = ops.kv4_cache(2, n_pages, n_seqs, max_pages, 1, 64), orc.Pages(n_pages, n_seqs, max_pages)
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache.pages.random_(0, 256, generator=g)
    shadow = cache.pages.clone()
    for _ in range(25):
        n = rng.randint(1, min(2 * n_seqs, 150))
        pick = lambda: [rng.randint(-1, n_seqs) if rng.random() < 0.1 else rng.randrange(n_seqs) for _ in range(n)]
        what = rng.choice(["extend", "extend", "fork", "free", "compact"])
        if what == "extend":
            s, c = pick(), [rng.choice([0, 1, 63, 64, 65, rng.randint(0, 20 * max_pages), -1 if rng.random() < 0.2 else 5]) for _ in range(n)]
            assert ops.kv4_extend(cache, dev(s), dev(c)).tolist() == model.extend(s, c)
        elif what == "fork":
            s, d = pick(), pick()
            assert ops.kv4_fork(cache, dev(s), dev(d)).tolist() == model.fork(s, d)
        elif what == "free":
            s = pick()[: max(1, n // 3)]
            ops.kv4_free(cache, dev(s))
            model.free(s)
        else:
            assert ops.kv4_compact(cache).tolist() == [model.compact()]
        for a, b in model.copied:
            shadow[:, b] = shadow[:, a]
        model.copied.clear()
        model.check(cache)
        assert torch.equal(cache.pages, shadow)


# ------------------------------------------------------------------------------------------------- all of them together
@pytest.mark.gpu
def test_a_server_with_a_layer_in_4_bits(built_lib):
    """A prompt in pieces, forked answers that go their own ways, one that leaves, compaction, further tokens: every token's layer (4-bit q | k | v product, rows into
    the cache, attention, 4-bit out-projection) against the same in 64 bits over what the cache holds of it."""
    rand = Rand(11)
    hidden, heads, kv_heads, dim, layers = 256, 4, 2, 64, 2
    width = (heads + 2 * kv_heads) * dim
    w_in = [ops.w4_quantize(rand(width, hidden, spread=hidden ** -0.5)) for _ in range(layers)]
    w_out = [ops.w4_quantize(rand(hidden, heads * dim, spread=(heads * dim) ** -0.5), group=32, symmetric=False) for _ in range(layers)]
    cache = ops.kv4_cache(layers, 40, 6, 12, kv_heads, dim)
    history = {0: [[] for _ in range(layers)]}   # what each sequence's cache holds, row by row

    def step(seqs, counts):
        rows = sum(counts)
        pos = ops.kv4_extend(cache, dev(seqs), dev(counts))
        first = pos.tolist()
        assert min(first) >= 0
        x = rand(rows, hidden)
        for layer in range(layers):
            p = ops.linear_w4(x, w_in[layer])
            q, k, v = (t.unflatten(1, (-1, dim)) for t in p.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
            where = (dev(seqs), starts_of(counts), pos)
            ops.kv4_store(cache, layer, k, v, *where)
            a = ops.kv4_attention(cache, layer, q, *where)
            row = 0
            for s, c, f in zip(seqs, counts, first):
                mine = history[s][layer]
                mine.extend(zip(orc.held(k[row:row + c]), orc.held(v[row:row + c])))
                assert len(mine) == f + c
                keys, values = (torch.stack([r[i] for r in mine]) for i in (0, 1))
                want, bound = orc.attention(q[row:row + c], keys, values, f, dim ** -0.5, 0)
                assert bool(((a[row:row + c].cpu().double() - want).abs() <= bound).all()), (s, layer, f)
                row += c
            x = ops.add(x, ops.linear_w4(a.flatten(1), w_out[layer]))
        return x

    step([0], [70])
    step([0], [1])
    step([0], [35])
    assert ops.kv4_fork(cache, dev([0, 0, 0]), dev([1, 2, 5])).tolist() == [1, 1, 1]
    for s in (1, 2, 5):
        history[s] = [list(h) for h in history[0]]
    step([1, 2, 5, 0], [1, 1, 1, 1])
    step([5, 0, 2, 1], [2, 30, 1, 1])
    ops.kv4_free(cache, dev([0, 2]))
    live = int(ops.kv4_compact(cache))
    assert live == int((cache.refs > 0).sum()) and not bool((cache.refs[live:] > 0).any())
    step([1, 5], [1, 40])
    history[3] = [[] for _ in range(layers)]
    step([3, 1], [130, 1])
