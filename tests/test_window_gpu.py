"""Windowed lane attention: against softmax in 64 bits over the keys that a row may see, bit by bit against itself (alone, among others,
serial), and where keys that nobody may see hold anything at all."""

import math

import pytest
import torch

from tests.helpers import assert_same_bits

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
CHUNK = 128


def make(seed, lens, widths, h, hk, d, extra_rows=0, fill=None):
    """Pages in shuffled order, stale rows and unowned pages filled with ``fill``."""

    gen = torch.Generator().manual_seed(seed)
    pages = [-(-(n + w) // 16) for n, w in zip(lens, widths)]
    count = sum(pages) + 2
    order = torch.randperm(count, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(max(pages), 1) + 1), -7, dtype=torch.int32)
    k, v = (torch.randn((count, hk, 16, d), generator=gen).to(BF) for _ in range(2))
    live = torch.zeros((count, 16), dtype=torch.bool)
    at = 0
    for s, n in enumerate(pages):
        table[s, :n] = order[at:at + n]
        for j in range(lens[s]):
            live[order[at + j // 16], j % 16] = True
        at += n
    if fill is not None:
        k.masked_fill_(~live[:, None, :, None], fill)
        v.masked_fill_(~live[:, None, :, None], fill)
    r = sum(widths) + extra_rows
    q, k_new, v_new = 2 * torch.randn((r, h, d), generator=gen), torch.randn((r, hk, d), generator=gen), torch.randn((r, hk, d), generator=gen)
    starts = [0]
    for w in widths:
        starts.append(starts[-1] + w)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    return dict(q=q.to(BF), k_new=k_new.to(BF), v_new=v_new.to(BF), k=k, v=v, table=table, lens=i32(lens), start=i32(starts))


def attend(c, lens, widths, window, sinks, chunk=CHUNK, context=None, **kw):
    from tensorfold_b200 import _lib, lane_window

    g = {n: t.cuda() for n, t in c.items()}
    lse = torch.full(c["q"].shape[:2], 77.0, device="cuda")
    out = kw.pop("out", torch.full_like(g["q"], 55.0))
    res = lane_window.window_attention(g["q"], g["k_new"], g["v_new"], g["k"], g["v"], g["table"], g["lens"], g["start"],
                                       scale=c["q"].shape[-1] ** -0.5, max_window=max(max(widths), 1), max_context=context or max(n + w for n, w in zip(lens, widths)),
                                       window=window, sinks=sinks, chunk_keys=chunk, lse=lse, out=out, **kw)
    torch.cuda.synchronize()
    _lib.status(g["q"].device).raise_if_set()
    return res if out is None else out, lse


def plain(c, s, lens, widths, window, sinks):
    """Outputs, log-sum-exps and the size of the terms of each row of sequence s, 64 bits."""

    d, hk = c["q"].shape[-1], c["k_new"].shape[1]
    g = c["q"].shape[1] // hk
    r0, n, w = int(c["start"][s]), lens[s], widths[s]
    used = c["table"][s, :-(-n // 16)].long()
    flat = lambda t: t[used].permute(0, 2, 1, 3).reshape(-1, hk, d)[:n]
    keys = torch.cat([flat(c["k"]), c["k_new"][r0:r0 + w]]).double().repeat_interleave(g, 1)
    vals = torch.cat([flat(c["v"]), c["v_new"][r0:r0 + w]]).double().repeat_interleave(g, 1)
    out, lse, size = [], [], []
    for t in range(w):
        p = n + t
        see = [j for j in range(p + 1) if window is None or p - j < window or j < sinks]
        sc = torch.einsum("hd,jhd->hj", c["q"][r0 + t].double(), keys[see]) * d ** -0.5
        pr = torch.softmax(sc, 1)
        out.append(torch.einsum("hj,jhd->hd", pr, vals[see]))
        size.append(torch.einsum("hj,jhd->hd", pr, vals[see].abs()))
        lse.append(torch.logsumexp(sc, 1))
    return torch.stack(out), torch.stack(lse), torch.stack(size)


def check(c, got, lse, lens, widths, window, sinks):
    for s in range(len(lens)):
        if not widths[s]:
            continue
        r0 = int(c["start"][s])
        want, wl, size = plain(c, s, lens, widths, window, sinks)
        g, l = got[r0:r0 + widths[s]].double().cpu(), lse[r0:r0 + widths[s]].double().cpu()
        # output: the weights are rounded to bf16 before the product (2^-8 of each term) and the result once (2^-8 of it); fp32 sums
        # of up to 256 products of size |q||k| scale ~ 2 * 16 / 2 put a score off by less than 2^-14, a weight by as much of itself
        bound = (2.0 ** -8 + 2.0 ** -12) * size + 2.0 ** -8 * want.abs()
        assert bool(((g - want).abs() <= bound).all()), (s, float(((g - want).abs() - bound).max()))
        # a score's error goes into the log-sum-exp as it is; its own rounding is 2^-23 of at most 64
        assert bool(((l - wl).abs() <= 2.0 ** -13).all()), (s, float((l - wl).abs().max()))


SHAPES = [(24, 4, 256), (16, 2, 128), (16, 1, 256), (3, 3, 128), (6, 1, 256)]


@pytest.mark.parametrize("h,hk,d", SHAPES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (64, 4), (100, 16), (257, 1), (130, 70), (5000, 4)])
def test_against_64_bits(lib, h, hk, d, window, sinks):
    lens, widths = [0, 1, 700, 15, 16, 129, 300, 640], [1, 3, 8, 0, 1, 2, 5, 1]
    c = make(h + d, lens, widths, h, hk, d)
    got, lse = attend(c, lens, widths, window, sinks)
    check(c, got, lse, lens, widths, window, sinks)


@pytest.mark.parametrize("h,hk,d", [(24, 4, 256), (16, 2, 128), (16, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (90, 5), (300, 0)])
def test_long_windows(lib, h, hk, d, window, sinks):
    """More query rows than one block takes, keys that are mostly the window's own, rows that stop seeing what the first ones saw."""

    lens, widths = [37, 0, 210], [211, 65, 128]
    c = make(3 * h, lens, widths, h, hk, d)
    got, lse = attend(c, lens, widths, window, sinks)
    check(c, got, lse, lens, widths, window, sinks)


@pytest.mark.parametrize("chunk", [64, 192, 512, 4096])
def test_other_chunks(lib, chunk):
    lens, widths = [1000, 63, 64, 517], [4, 1, 1, 8]
    c = make(chunk, lens, widths, 24, 4, 256)
    for window, sinks in ((None, 0), (200, 70)):
        got, lse = attend(c, lens, widths, window, sinks, chunk=chunk, context=1100)
        check(c, got, lse, lens, widths, window, sinks)


@pytest.mark.parametrize("h,hk,d", [(24, 4, 256), (16, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (130, 4), (64, 20)])
def test_a_chunk_a_row_gives_the_bits_of_the_join(lib, h, hk, d, window, sinks):
    """max_context decides whether there is one slot, and with it the way the results take."""

    lens, widths = [400, 3, 0, 77, 511], [9, 140, 1, 0, 1]
    c = make(41, lens, widths, h, hk, d, extra_rows=2)
    one, lse = attend(c, lens, widths, window, sinks, chunk=512, context=512)
    two, lse2 = attend(c, lens, widths, window, sinks, chunk=512, context=513)
    assert_same_bits(one, two)
    assert_same_bits(lse, lse2)
    assert bool((one[-2:] == 55).all()) and bool((lse[-2:] == 77).all())
    check(c, one, lse, lens, widths, window, sinks)


@pytest.mark.parametrize("h,hk,d", [(24, 4, 256), (16, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (130, 4), (64, 20)])
def test_a_window_has_the_bits_of_serial_steps(lib, h, hk, d, window, sinks):
    lens, widths = [500, 121, 9], [8, 7, 8]
    c = make(7, lens, widths, h, hk, d)
    got, lse = attend(c, lens, widths, window, sinks, context=600)
    for s, n in enumerate(lens):
        r0 = int(c["start"][s])
        for t in range(widths[s]):
            one = dict(c, table=c["table"][s:s + 1].contiguous(), lens=torch.tensor([n + t], dtype=torch.int32), start=torch.tensor([0, 1], dtype=torch.int32))
            for name in ("q", "k_new", "v_new"):
                one[name] = c[name][r0 + t:r0 + t + 1].contiguous()
            one["k"], one["v"] = c["k"].clone(), c["v"].clone()
            for j in range(n, n + t):                   # rows 0..t-1 are committed by now
                page = int(c["table"][s, j // 16])
                one["k"][page, :, j % 16] = c["k_new"][r0 + j - n]
                one["v"][page, :, j % 16] = c["v_new"][r0 + j - n]
            alone, l1 = attend(one, [n + t], [1], window, sinks, context=600)
            assert_same_bits(alone, got[r0 + t:r0 + t + 1], f"sequence {s} row {t}")
            assert_same_bits(l1, lse[r0 + t:r0 + t + 1], f"lse of sequence {s} row {t}")


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38])
def test_keys_that_nobody_sees_may_hold_anything(lib, bad):
    """Stale rows behind the committed length, pages outside the window, unowned pages, and later rows of the same window."""

    lens, widths = [700, 33, 5], [8, 3, 2]
    window, sinks = 120, 4
    clean = make(5, lens, widths, 24, 4, 256)
    want, wl = attend(clean, lens, widths, window, sinks)
    c = make(5, lens, widths, 24, 4, 256, fill=bad)
    for s, n in enumerate(lens):
        for j in range(sinks, max(sinks, n + 1 - window)):
            c["k"][int(c["table"][s, j // 16]), :, j % 16] = bad
            c["v"][int(c["table"][s, j // 16]), :, j % 16] = bad
        for i in range(-(-sinks // 16), max(0, n + 1 - window) // 16):
            c["table"][s, i] = 2 ** 30                       # given back: not followed
    got, lse = attend(c, lens, widths, window, sinks)
    assert_same_bits(got, want)
    assert_same_bits(lse, wl)
    for s in range(3):                                       # the last row of each window is bad: the rows before it do not see it
        at = int(c["start"][s + 1]) - 1
        c["k_new"][at] = bad
        c["v_new"][at] = bad
    got, lse = attend(c, lens, widths, window, sinks)
    for s in range(3):
        part = slice(int(c["start"][s]), int(c["start"][s + 1]) - 1)
        assert_same_bits(got[part], want[part])
        assert_same_bits(lse[part], wl[part])
    # and a key that has left the window of all rows but the first is not seen by the others
    c = make(5, lens, widths, 24, 4, 256)
    j = 700 + 1 - window
    c["v"][int(c["table"][0, j // 16]), :, j % 16] = bad
    c["k"][int(c["table"][0, j // 16]), :, j % 16] = bad
    got, lse = attend(c, lens, widths, window, sinks)
    assert_same_bits(got[1:8], want[1:8])
    assert_same_bits(lse[1:], wl[1:])


def test_rows_behind_the_last_sequence_are_left(lib):
    lens, widths = [100, 40], [3, 2]
    c = make(9, lens, widths, 24, 4, 256, extra_rows=4)
    got, lse = attend(c, lens, widths, 64, 4)
    check(c, got, lse, lens, widths, 64, 4)
    assert bool((got[5:] == 55).all()) and bool((lse[5:] == 77).all())


@pytest.mark.parametrize("group", [64, 32])
@pytest.mark.parametrize("h,hk,d", [(24, 4, 256), (16, 2, 128)])
def test_gate_and_packed_output(lib, h, hk, d, group):
    from tensorfold_b200 import lane_qmm

    lens, widths = [200, 0, 77], [5, 1, 3]
    c = make(11, lens, widths, h, hk, d)
    r = sum(widths)
    proj = torch.randn((r, 2 * h * d + 64), generator=torch.Generator().manual_seed(1)).to(BF).cuda()[:, :2 * h * d]
    out, _ = attend(c, lens, widths, 100, 4)
    packed = lane_qmm.new_packed(r, h * d, group, "cuda")
    packed.data.fill_(0xFF)
    gated, _ = attend(c, lens, widths, 100, 4, gate=proj, packed_out=packed)
    plain_gate = (out.float() * torch.sigmoid(proj.float().reshape(r, h, 2, d)[:, :, 1])).to(BF)
    # the kernel's sigmoid is off by a few units in 2^-24: at most one bf16 step where the product is near a border
    assert bool(((gated.float() - plain_gate.float()).abs() <= 2.0 ** -8 * plain_gate.float().abs()).all())
    assert torch.equal(packed.data, lane_qmm.pack_rows(gated.reshape(r, h * d), group).data)


def test_capture_another_stream_and_no_scratch_of_its_own(lib):
    from tensorfold_b200 import lane_window

    lens, widths = [900, 30], [4, 8]
    c = {n: t.cuda() for n, t in make(13, lens, widths, 24, 4, 256).items()}
    kw = dict(scale=1 / 16, max_window=8, max_context=1000, window=300, sinks=4, chunk_keys=128)
    args = (c["q"], c["k_new"], c["v_new"], c["k"], c["v"], c["table"], c["lens"], c["start"])
    want = lane_window.window_attention(*args, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = lane_window.window_attention(*args, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert_same_bits(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = lane_window.window_attention(*args, **kw)
    c["q"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert_same_bits(held, lane_window.window_attention(*args, **kw))


def test_reports_and_refusals(lib):
    from tensorfold_b200 import _lib, lane_window

    lens, widths = [100], [2]
    c = {n: t.cuda() for n, t in make(15, lens, widths, 24, 4, 256).items()}
    args = [c["q"], c["k_new"], c["v_new"], c["k"], c["v"], c["table"], c["lens"], c["start"]]
    kw = dict(scale=1 / 16, max_window=2, max_context=102)
    lane_window.window_attention(*args, **kw)
    status = _lib.status(c["q"].device)
    status.raise_if_set()
    for changed in (dict(scale=0.0), dict(scale=math.inf), dict(window=0), dict(sinks=-1), dict(max_window=0), dict(max_context=1), dict(chunk_keys=100),
                    dict(chunk_keys=0), dict(lse=torch.empty((2, 24), dtype=BF, device="cuda")), dict(out=torch.empty((2, 24, 128), dtype=BF, device="cuda")),
                    dict(scratch=torch.empty(16, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(ValueError):
            lane_window.window_attention(*args, **{**kw, **changed})
    for i, bad in ((0, c["q"].float()), (0, c["q"].transpose(0, 1)), (1, c["k_new"][:1]), (3, c["k"][:, :3]), (5, c["table"].long()), (6, c["lens"].cpu()),
                   (0, c["q"][:, :23].contiguous())):
        with pytest.raises(ValueError):
            lane_window.window_attention(*[bad if j == i else t for j, t in enumerate(args)], **kw)
    # a longer sequence than promised, and a page that is none: reported, nothing read out of range
    lane_window.window_attention(*args, **{**kw, "max_context": 64})
    with pytest.raises(RuntimeError):
        status.raise_if_set()
    c["table"][0, 1] = c["k"].shape[0]
    lane_window.window_attention(*args, **kw)
    with pytest.raises(RuntimeError):
        status.raise_if_set()


@pytest.mark.parametrize("h,hk,d", [(24, 4, 256), (8, 2, 128), (6, 1, 256)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (300, 4)])
def test_clusters_give_the_bits_of_the_join(lib, h, hk, d, window, sinks):
    """One sequence alone, whose chunks a cluster joins, and among many, whose chunks go through memory; gate and packed rows, with the padding."""

    from tensorfold_b200.lane_qmm import new_packed

    lens, widths = [700, 515, 130, 3, 900, 64, 257, 800, 31, 555], [2, 1, 2, 1, 2, 1, 2, 1, 2, 1]
    c = make(77, lens, widths, h, hk, d)
    got, lse = attend(c, lens, widths, window, sinks, context=1000)
    for s in range(len(lens)):
        r0, w = int(c["start"][s]), widths[s]
        one = dict(c, table=c["table"][s:s + 1].contiguous(), lens=c["lens"][s:s + 1].contiguous(), start=torch.tensor([0, w], dtype=torch.int32),
                   **{n: c[n][r0:r0 + w].contiguous() for n in ("q", "k_new", "v_new")})
        alone, lse1 = attend(one, lens[s:s + 1], [w], window, sinks, context=1000)
        assert_same_bits(alone, got[r0:r0 + w])
        assert_same_bits(lse1, lse[r0:r0 + w])
        # packed rows, by a cluster and (beside nineteen sequences without rows) by the join
        gate = torch.randn((w, h * 2 * d), generator=torch.Generator().manual_seed(s)).to(BF).cuda()
        packs = []
        for seqs in (1, 20):
            many = dict(one, table=one["table"].repeat(seqs, 1), lens=one["lens"].repeat(seqs), start=torch.tensor([0] + [w] * seqs, dtype=torch.int32))
            packed = new_packed(w, h * d, 64, "cuda")
            packed.data.fill_(7)
            attend(many, lens[s:s + 1] * seqs, [w], window, sinks, context=1000, out=None, gate=gate, packed_out=packed)
            packs.append(packed.data.clone())
        assert_same_bits(packs[0], packs[1])
