"""The paged cache of 4-bit keys and values where it can go wrong: windows behind all of a sequence whose row of the table is full, lengths that change while a
call runs, values that are no numbers behind weights of nothing."""
import re

import pytest
import torch

import kv4_oracle as orc
from test_kv4_gpu import Rand, dev, filled, starts_of
from tinygpt_b200 import build, ops
from tinygpt_b200._lib import B200Error

BF16 = torch.bfloat16


# ------------------------------------------------------------------------------------------------- full rows of the table
@pytest.mark.gpu
@pytest.mark.parametrize("pages,rows", [(1, 1), (3, 1), (300, 1), (300, 6), (3, 50), (40, 50)])   # clusters, the even cut, blocks for a CTA
def test_windows_behind_a_full_row(built_lib, pages, rows):
    """The last sequence fills its row of the table, which lies in front of other numbers; rows that see its last tokens or nothing."""
    rand, heads, dim, length = Rand(21), 4, 64, 64 * pages
    plain = ops.kv4_cache(1, 2 * pages + 4, 2, pages, 1, dim)
    numbers = torch.full((2 * pages + 8,), 2 * pages + 3, dtype=torch.int32, device="cuda")   # a page of NaN, behind the table
    numbers[:2 * pages] = torch.arange(2 * pages, device="cuda", dtype=torch.int32).flip(0)
    cache = ops.KV4Cache(plain.pages, numbers[:2 * pages].view(2, pages), plain.length, plain.refs, 1, dim)
    cache.pages.fill_(255)
    cache.refs[:2 * pages] = 1
    cache.length.copy_(dev([length, length]))
    k, v = rand(2 * length, 1, dim), rand(2 * length, 1, dim)
    ops.kv4_store(cache, 0, k, v, dev([0, 1]), dev([0, length, 2 * length]), dev([0, 0]))
    hk, hv, q = orc.held(k), orc.held(v), rand(2 * rows, heads, dim)
    for window in (1, 33, 64):
        for at in (length - rows, length, length + window - 1 - rows // 2, length + window - 2, length + window - 1, length + window, length + 5000):
            out = ops.kv4_attention(cache, 0, q, dev([0, 1]), dev([0, rows, 2 * rows]), dev([at, at]), window=window).cpu().double()
            for s in (0, 1):
                mine = slice(s * length, (s + 1) * length)
                want, bound = orc.attention(q[s * rows:(s + 1) * rows], hk[mine], hv[mine], at, dim ** -0.5, window)
                got = out[s * rows:(s + 1) * rows]
                assert bool(((got - want).abs() <= bound).all()), (window, at, s)
                blind = max(0, min(rows, at + rows - (length + window - 1)))
                assert blind == 0 or not got[rows - blind:].any()


# ------------------------------------------------------------------------------------------------- lengths that change
def test_what_warps_meet_by_is_read_once():
    """Another stream may write to a length while a call runs, and a warp that waits at a barrier for one that went by another length waits for good.  So the lists and
    the lengths are read in one place, the kernel whose warps go together goes by one reading, and no barrier's threads are counted by what was read.  (That warps that go
    alone come to an end by whatever they read is tests/test_kv4_steps.py's.)"""
    text = (build.CSRC / "kv4_attn.cu").read_text()
    body = text[text.index("kv4_read(const Kv4Attn& p, int i) {"):]
    body = body[:body.index("\n}\n")]
    for what in ("p.cache.length[", "p.pos[", "p.seqs["):
        assert text.count(what) == body.count(what) == 1, what
    # kv4_read by a thread of the plan, into shared memory, by a lane for its warp, and of lane 0 for a warp
    for what in ("EXACT ? rows[i] : kv4_read(p, i)", "[k] = kv4_read(p, k)", "EXACT ? rows[lane] : kv4_read(p, lane)", "kv4_read_warp(const Kv4Attn& p, int i) {"):
        assert text.count(what) == 1, what
    assert text.count("kv4_read(p, ") == 4 and text.count("kv4_read_warp(p, ") == 2
    assert "bar_sync" not in text and "barrier" not in re.sub(r"//.*", "", text)


# ------------------------------------------------------------------------------------------------- values that are no numbers
@pytest.mark.gpu
@pytest.mark.parametrize("rows,room", [(1, 1), (1, 9000), (7, 1), (7, 9000), (60, 1)])   # clusters, the even cut, one and two tiles; a CTA's block
@pytest.mark.parametrize("low", [(10, 11), (0, 32), (138, 139), (128, 160), (0, 160)])   # tokens with next to no weight: one of a step, a step, all that is in a piece
def test_a_value_that_is_seen_counts_whatever_its_weight(built_lib, rows, room, low):
    """A weight that is rounded to nothing makes nothing of a value that is not a number, whether the step is seen whole or in part and wherever it is joined."""
    rand, dim, length = Rand(23), 128, 161 + rows
    cache, seqs, k, v = filled(rand, [length], 2, dim, room=room)
    k.zero_()
    k[low[0]:low[1]] = -40.0
    v[low[0], 0, 5] = float("nan")
    ops.kv4_store(cache, 0, k, v, seqs, dev([0, length]), dev([0]))
    q = torch.ones(rows, 4, dim, device="cuda", dtype=BF16)
    for at in (length - rows, max(low[0] - rows // 2, 0)):
        out = ops.kv4_attention(cache, 0, q, seqs, dev([0, rows]), dev([at])).cpu().double()
        want, bound = orc.attention(q, orc.held(k), orc.held(v), at, dim ** -0.5, 0)
        assert torch.equal(out.isnan(), want.isnan()) and bool(want[-1, :2, :64].isnan().all())
        rest = ~want.isnan()
        assert bool(((out - want).abs() <= bound)[rest].all())


# ------------------------------------------------------------------------------------------------- calls of all kinds
@pytest.mark.gpu
def test_calls_without_a_sequence(built_lib):
    """A server's step in which no sequence lives: rows belong to nobody, whichever way the call goes (contiguous tensors, others)."""
    rand, none, start = Rand(24), dev([]), dev([0])
    cache, seqs, k, v = filled(rand, [70, 3], 2, 64)
    was = [t.clone() for t in (cache.pages, cache.table, cache.length, cache.refs)]
    wide = rand(5, 4, 64)
    for x in (wide[:, :2].contiguous(), wide[:, :2], wide.transpose(0, 1)[:2].transpose(0, 1)):
        assert ops.kv4_store(cache, 0, x, x, none, start, none) is None
        assert not ops.kv4_attention(cache, 0, x, none, start, none).any()
    for rows in (0, 5):
        got = ops.kv4_load(cache, 0, none, start, none, rows)
        assert all(t.shape == (rows, 2, 64) and t.dtype == torch.float32 and not t.any() for t in got)
    assert ops.kv4_extend(cache, none, none).shape == ops.kv4_fork(cache, none, none).shape == (0,) and ops.kv4_free(cache, none) is None
    assert all(torch.equal(a, b) for a, b in zip(was, (cache.pages, cache.table, cache.length, cache.refs)))


@pytest.mark.gpu
def test_numbers_past_64_bits_are_refused(built_lib):
    """On both ways, the native one and the one that other tensors take: none of them comes out as another layer or window."""
    rand = Rand(25)
    cache, seqs, k, v = filled(rand, [70, 3], 2, 64)
    where, wide = (seqs, dev([0, 1, 2]), dev([69, 2])), rand(2, 2, 64)
    for x in (wide, wide.transpose(1, 2).contiguous().transpose(1, 2)):
        assert ops.kv4_attention(cache, 0, x, *where, window=2 ** 62).isfinite().all()
        for bad in (2 ** 64, 2 ** 63, -1, 2 ** 64 + 1, -2 ** 64):
            for call in (lambda: ops.kv4_attention(cache, bad, x, *where), lambda: ops.kv4_attention(cache, 0, x, *where, window=bad),
                         lambda: ops.kv4_store(cache, bad, x, x, *where), lambda: ops.kv4_load(cache, bad, *where, 2)):
                with pytest.raises(B200Error):
                    call()


# ------------------------------------------------------------------------------------------------- numbers up to the stated bounds
@pytest.mark.gpu
@pytest.mark.parametrize("rows,room", [(1, 1), (1, 9000), (7, 9000), (60, 1)])
@pytest.mark.parametrize("dim", [64, 256])
def test_numbers_up_to_the_stated_bounds(built_lib, rows, room, dim):
    """Queries of one sign just below 2^112 over keys of one sign, values of one sign whose sum over the tokens comes to 2^118 and weights that rise to almost 2^8
    above the running maximum: everything stays finite, and right."""
    rand, length = Rand(26), 1023
    cache, seqs, k, v = filled(rand, [length], 1, dim, room=room)
    up = torch.linspace(0.5, 0.96, length, device="cuda")[:, None, None] * (1 + 0.02 * torch.rand(length, 1, dim, generator=rand.g, device="cuda"))
    k = up.to(BF16)
    v = ((1 - 0.5 * torch.rand(length, 1, dim, generator=rand.g, device="cuda")) * 2.0 ** 108).to(BF16).clamp(max=2.0 ** 108 * (1 - 2.0 ** -8))
    v[::2, :, :64] = v[0, :, :1]   # groups of one number beside others
    ops.kv4_store(cache, 0, k, v, seqs, dev([0, length]), dev([0]))
    q = torch.full((rows, 4, dim), 2.0 ** 112 * (1 - 2.0 ** -8), device="cuda").to(BF16)
    scale = 12.0 / dim * 2.0 ** -112   # scores from 6 to some 11.6: 2^8 in weight
    out = ops.kv4_attention(cache, 0, q, seqs, dev([0, rows]), dev([length - rows]), scale=scale).cpu().double()
    want, bound = orc.attention(q, orc.held(k), orc.held(v), length - rows, scale, 0)
    assert bool(torch.isfinite(out).all()) and bool(((out - want).abs() <= bound).all())
    # and with queries of the other sign, whose scores fall
    out = ops.kv4_attention(cache, 0, -q, seqs, dev([0, rows]), dev([length - rows]), scale=scale).cpu().double()
    want, bound = orc.attention(-q, orc.held(k), orc.held(v), length - rows, scale, 0)
    assert bool(torch.isfinite(out).all()) and bool(((out - want).abs() <= bound).all())


def test_parts_of_a_cache_are_checked(built_lib):
    """A cache put together from tensors at hand: kernels take its sizes from them, so what does not fit is refused."""
    page = 2 * 64 * (64 // 2 + 4)
    ok = dict(pages=torch.empty(1, 4, page, dtype=torch.uint8), table=torch.zeros(2, 3, dtype=torch.int32), length=torch.zeros(2, dtype=torch.int32),
              refs=torch.zeros(4, dtype=torch.int32), kv_heads=1, head_dim=64)
    for bad, what in ((dict(pages=ok["pages"].float()), "pages"), (dict(pages=ok["pages"][0]), "pages"), (dict(pages=ok["pages"][..., :-1]), "pages"),
                      (dict(table=ok["table"].long()), "table"), (dict(table=ok["table"].t()), "table"), (dict(table=ok["table"][0]), "table"),
                      (dict(length=ok["length"][:1]), "length"), (dict(refs=ok["refs"][:3]), "refs"), (dict(refs=ok["refs"].float()), "refs"),
                      (dict(head_dim=128), "pages"), (dict(head_dim=32), "heads"), (dict(kv_heads=0), "heads"), ({}, "CUDA device")):
        with pytest.raises(B200Error, match=what):
            ops.KV4Cache(**{**ok, **bad})


@pytest.mark.gpu
@pytest.mark.parametrize("rows,room", [(1, 1), (1, 9000), (7, 9000), (60, 1)])
def test_a_window_over_everything_masks_nothing(built_lib, rows, room):
    rand, length = Rand(27), 300
    cache, seqs, k, v = filled(rand, [length], 2, 64, room=room)
    q = rand(rows, 4, 64)
    args = (cache, 0, q, seqs, dev([0, rows]), dev([length - rows]))
    want = ops.kv4_attention(*args)
    for window in (length, 2 ** 30, 2 ** 31 - 65, 2 ** 31 - 32, 2 ** 31 - 1, 2 ** 31, 2 ** 62):
        assert torch.equal(ops.kv4_attention(*args, window=window), want), window


@pytest.mark.gpu
@pytest.mark.parametrize("rows,room", [(5, 1), (5, 9000), (12, 9000), (60, 1), (150, 1)])
@pytest.mark.parametrize("dim", [64, 256])
def test_masked_numbers_that_are_none(built_lib, rows, room, dim):
    """Keys and values that are not finite, behind a row's own position and in front of its window, change nothing for that row, in every way; for rows that see them
    they count."""
    rand, length, window = Rand(28), 333, 90
    cache, seqs, k, v = filled(rand, [length], 2, dim, room=room)
    q, first = rand(rows, 4, dim), length - rows
    args = (cache, 0, q, seqs, dev([0, rows]), dev([first]))
    plain, windowed = ops.kv4_attention(*args), ops.kv4_attention(*args, window=window)
    for t in (first + rows // 2, first, length - 1, first - 10, max(first + rows // 2 - window, 0)):
        for which in (0, 1):
            bad = [x[t:t + 1].clone() for x in (k, v)]
            bad[which][0, :, 3::64] = (float("nan"), float("inf"))[t % 2]
            ops.kv4_store(cache, 0, *bad, seqs, dev([0, 1]), dev([t]))
            for got, want, w in ((ops.kv4_attention(*args), plain, 0), (ops.kv4_attention(*args, window=window), windowed, window)):
                at = first + torch.arange(rows)
                sees = (at >= t) & ((at - t < w) | (w == 0))
                assert torch.equal(got.cpu()[~sees], want.cpu()[~sees]) and bool(got.cpu()[sees].isnan().all()), (t, which, w)
            ops.kv4_store(cache, 0, k[t:t + 1], v[t:t + 1], seqs, dev([0, 1]), dev([t]))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,room", [(1, 1), (1, 9000), (7, 9000), (60, 1)])
def test_positions_to_the_end_of_32_bits(built_lib, rows, room):
    """Rows far behind what the sequence holds see of it what their window reaches."""
    rand, length = Rand(29), 300
    cache, seqs, k, v = filled(rand, [length], 2, 64, room=room)
    q, hk, hv = rand(rows, 4, 64), orc.held(k), orc.held(v)
    for at in (2 ** 30 - 1, 2 ** 30 + 7, 2 ** 31 - 300, 2 ** 31 - 70 - rows):
        for back in (1, 31, 200, length - 1 + rows, length + 500):   # the first row's window ends so far behind the first token
            window = at - back
            want, bound = orc.attention(q, hk, hv, at, 64 ** -0.5, window)
            got = ops.kv4_attention(cache, 0, q, seqs, dev([0, rows]), dev([at]), window=window).cpu().double()
            assert bool(((got - want).abs() <= bound).all()), (at, back)


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 9000])
def test_a_sequence_twice_in_a_call(built_lib, room):
    """Two pieces of one sequence, stored and attended in one call: places in one tile of 16 and apart."""
    rand, heads, dim = Rand(30), 4, 64
    cache = ops.kv4_cache(1, 8, 2, 4 + room, 2, dim)
    cache.pages.fill_(255)
    assert ops.kv4_extend(cache, dev([1, 0]), dev([200, 70])).tolist() == [0, 0]
    k, v, q = rand(270, 2, dim), rand(270, 2, dim), rand(270, heads, dim)
    # rows: of sequence 1 positions 0 … 7, of it 8 … 99, of sequence 0 all, of sequence 1 100 … 199
    seqs, starts, pos = dev([1, 1, 0, 1]), dev([0, 8, 100, 170, 270]), dev([0, 8, 0, 100])
    ops.kv4_store(cache, 0, k, v, seqs, starts, pos)
    for got, x in zip(ops.kv4_load(cache, 0, seqs, starts, pos, 270), (k, v)):
        assert torch.equal(got.cpu(), orc.held(x))
    hk, hv = ({1: torch.cat((orc.held(x)[:100], orc.held(x)[170:])), 0: orc.held(x)[100:170]} for x in (k, v))
    for rows, at in ([(0, 8), (8, 100), (100, 170), (170, 270)], [0, 8, 0, 100]), ([(7, 8), (99, 100), (169, 170), (269, 270)], [7, 99, 69, 199]):
        x = torch.cat([q[a:b] for a, b in rows])
        counts = [b - a for a, b in rows]
        out, row = ops.kv4_attention(cache, 0, x, seqs, starts_of(counts), dev(at)).cpu().double(), 0
        for s, c, p in zip((1, 1, 0, 1), counts, at):
            want, bound = orc.attention(x[row:row + c], hk[s], hv[s], p, dim ** -0.5, 0)
            assert bool(((out[row:row + c] - want).abs() <= bound).all()), (s, c, p)
            row += c


@pytest.mark.gpu
def test_calls_on_several_streams(built_lib):
    """Calls of every way at once, each with its own workspace, over one cache that none of them writes, beside Linears of every way."""
    rand, dim = Rand(31), 128
    lengths = [3000, 64, 700, 1111]
    big, seqs, _, _ = filled(rand, lengths, 2, dim, room=9000)
    small, few, _, _ = filled(rand, [900, 33], 2, dim)
    w = ops.w4_quantize(rand(512, 1024, spread=0.03))
    jobs = []
    for cache, s, ls in ((big, seqs, lengths), (small, few, [900, 33])):
        for rows in (1, 6, 60):
            counts = [min(rows, l) for l in ls]
            q, st, pos = rand(sum(counts), 4, dim), starts_of(counts), dev([l - c for l, c in zip(ls, counts)])
            jobs.append(lambda cache=cache, q=q, s=s, st=st, pos=pos: ops.kv4_attention(cache, 0, q, s, st, pos))
    for m in (1, 20, 100, 300):
        x = rand(m, 1024)
        jobs.append(lambda x=x: ops.linear_w4(x, w))
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for turn in range(20):
        for n, st in enumerate(streams):
            with torch.cuda.stream(st):
                for i in range(len(jobs)):
                    j = (i * (2 * n + 1) + turn) % len(jobs)
                    got.append((j, jobs[j]()))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[j]) for j, y in got)


class Guarded:
    """Device memory between two guards; what it held before is numbers that are none."""

    def __init__(self, nbytes):
        self.all = torch.full((4096 + -(-nbytes // 256) * 256 + 4096,), 255, dtype=torch.uint8, device="cuda")
        self.at, self.nbytes = self.all.data_ptr() + 4096, nbytes

    def view(self, dtype, *shape):
        return self.all[4096:4096 + self.nbytes].view(dtype).view(shape)

    def intact(self):
        return bool((self.all[:4096] == 255).all()) and bool((self.all[4096 + self.nbytes:] == 255).all())


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,counts,heads,kv_heads,dim,room", [([900, 33], [1, 1], 14, 2, 64, 0), ([3000, 64, 700], [1, 1, 1], 24, 8, 128, 9000), ([700] * 40, [1] * 40, 4, 2, 64, 9000),
                                                                    ([3000, 300], [6, 20], 4, 2, 256, 9000), ([900, 300], [257, 1], 16, 8, 128, 0), ([500], [200], 4, 1, 192, 0),
                                                                    ([60] * 40, [50] * 40, 4, 2, 64, 0)])
def test_calls_of_the_library_stay_within_their_memory(built_lib, lengths, counts, heads, kv_heads, dim, room):
    """The C entry points with workspaces and results of just the bytes they ask for, whatever those held before."""
    import ctypes as C
    from tinygpt_b200._lib import lib
    rand, n, rows = Rand(32), len(lengths), sum(counts)
    cache, seqs, k, v = filled(rand, lengths, kv_heads, dim, room=room)
    d, stream = C.byref(cache._desc), torch.cuda.current_stream().cuda_stream
    q, st, pos = rand(rows, heads, dim), starts_of(counts), dev([l - c for l, c in zip(lengths, counts)])
    want = ops.kv4_attention(cache, 0, q, seqs, st, pos)
    out, ws = Guarded(2 * q.numel()), Guarded(lib().b200_kv4_attention_workspace_bytes(d, heads, n, rows))
    assert lib().b200_kv4_attention(out.at, q.data_ptr(), heads * dim, d, 0, heads, seqs.data_ptr(), st.data_ptr(), pos.data_ptr(), n, rows, dim ** -0.5, 0,
                                    ws.at if ws.nbytes else None, stream) == 0
    assert torch.equal(out.view(BF16, *q.shape), want) and out.intact() and ws.intact()
    total = sum(lengths)
    keys, vals = Guarded(4 * k.numel()), Guarded(4 * v.numel())
    assert lib().b200_kv4_load(keys.at, vals.at, d, 0, seqs.data_ptr(), starts_of(lengths).data_ptr(), dev([0] * n).data_ptr(), n, total, stream) == 0
    assert torch.equal(vals.view(torch.float32, *v.shape).cpu(), orc.held(v)) and keys.intact() and vals.intact()
    ws = Guarded(lib().b200_kv4_workspace_bytes(d))
    for call, other in (("extend", [64] * n), ("fork", [n] * n)):
        got, others = Guarded(4 * n), dev(other)
        assert getattr(lib(), f"b200_kv4_{call}")(d, seqs.data_ptr(), others.data_ptr(), got.at, n, ws.at, stream) == 0
        assert got.intact() and ws.intact()
    live = Guarded(4)
    assert lib().b200_kv4_free(d, seqs.data_ptr(), n // 2 + 1, stream) == 0 and lib().b200_kv4_compact(d, live.at, ws.at, stream) == 0
    assert int(live.view(torch.int32, 1)) == int((cache.refs > 0).sum()) and live.intact() and ws.intact()
