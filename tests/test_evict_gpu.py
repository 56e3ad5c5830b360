"""Attention weight per cached key, and eviction by it: against 64 bits, slot by slot, and through rounds of both."""

import math

import pytest
import torch

from tests.helpers import assert_same_bits

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
i32 = lambda x: torch.tensor(x, dtype=torch.int32)


def cache(seed, layers, lens, hk, d, spare=2):
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // 16) for n in lens]
    count = sum(need) + spare
    order = torch.randperm(count, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -3, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    k, v = (torch.randn((layers, count, hk, 16, d), generator=gen).to(BF) for _ in range(2))
    mass = torch.rand((layers, count, hk, 16), generator=gen) ** 3
    pos = torch.randint(0, 1 << 20, (layers, count, hk, 16), generator=gen).to(torch.int32)
    return table, k, v, mass, pos, gen


def cells(table, s, n):
    j = torch.arange(n)
    return table[s].long()[j // 16], j % 16


@pytest.mark.parametrize("h,hk,d", [(24, 4, 256), (16, 2, 128), (16, 1, 256), (5, 5, 128)])
@pytest.mark.parametrize("long_rows", [False, True])
def test_mass_against_64_bits(lib, h, hk, d, long_rows):
    from tensorfold_b200 import _lib, lane_evict

    layers, g = 2, h // hk
    lens, widths, keep = ([0, 40, 300], [33, 60, 128], [30, 60, 101]) if long_rows else ([0, 1, 15, 16, 300, 127, 128, 500], [1, 2, 8, 1, 5, 3, 0, 8], [1, 2, 8, 0, 3, 3, 0, 1])
    table, k, _, mass, pos, gen = cache(h, layers, [n + w for n, w in zip(lens, widths)], hk, d)
    r = sum(widths) + 3
    q = (2 * torch.randn((layers, r, h, d), generator=gen)).to(BF)
    lse = 6 + 2 * torch.rand((layers, r, h), generator=gen)
    row_pos = torch.randint(0, 10000, (r,), generator=gen).to(torch.int32)
    start = [0]
    for w in widths:
        start.append(start[-1] + w)
    want_m, want_p, size = mass.double(), pos.clone(), torch.zeros(mass.shape, dtype=torch.float64)
    for s, (n, m) in enumerate(zip(lens, keep)):
        if not m:
            continue
        pg, pl = cells(table, s, n + m)
        for layer in range(layers):
            keys = k[layer, pg, :, pl].double()                                 # [slots, hk, d]
            rows = slice(start[s], start[s] + m)
            sc = torch.einsum("tkgd,jkd->kgtj", q[layer, rows].double().reshape(m, hk, g, d), keys) * d ** -0.5
            e = (sc - lse[layer, rows].double().reshape(m, hk, g).permute(1, 2, 0).unsqueeze(-1)).exp()
            e = e.masked_fill(torch.arange(n + m) > torch.arange(n, n + m).unsqueeze(1), 0.0).sum((1, 2))    # [hk, slots]
            old = want_m[layer, pg, :, pl].T.clone()
            old[:, n:] = 0.0
            want_m[layer, pg, :, pl] = (old + e).T
            size[layer, pg, :, pl] = (old + e).T
            want_p[layer, pg[n:], :, pl[n:]] = row_pos[start[s]:start[s] + m].reshape(m, 1).expand(m, hk)
    dm, dp = mass.cuda(), pos.cuda()
    lane_evict.attention_mass(q.cuda(), lse.cuda(), k.cuda(), table.cuda(), i32(lens).cuda(), i32(start).cuda(), i32(keep).cuda(), row_pos.cuda(), dm, dp,
                              scale=d ** -0.5, max_window=max(widths), max_context=max(n + w for n, w in zip(lens, widths)))
    _lib.status(dm.device).raise_if_set()
    # a score off by less than 2^-14 (fp32 sums of 256 products) puts its weight off by that much of itself; the sum of up to
    # 128 x 16 positive terms in fp32 by less than 2^-13 of itself
    err = (dm.double().cpu() - want_m).abs()
    assert bool((err <= 2.0 ** -12 * size).all()), float((err - 2.0 ** -12 * size).max())
    assert torch.equal(dp.cpu(), want_p)                                        # nothing else is written


def select(mass, pos, n, budget, recent, sinks, nxt):
    """Kept slots of one (layer, sequence, head): protected, then by mass, ties to the lower slot."""

    key = [(0 if p < sinks or p >= nxt - recent else 1, -(m if m == m else -math.inf), j) for j, (m, p) in enumerate(zip(mass, pos))][:n]
    kept = sorted(j for *_, j in sorted(key)[:budget])
    holes = sorted(set(range(budget)) - set(kept))
    return holes, [j for j in kept if j >= budget]


@pytest.mark.parametrize("hk,d", [(4, 256), (2, 128), (1, 256)])
@pytest.mark.parametrize("kind", ["plain", "ties", "zeros", "strange"])
@pytest.mark.parametrize("budget,recent,sinks", [(100, 16, 4), (64, 64, 0), (1, 0, 0), (333, 0, 5), (40, 10, 0)])
def test_evict_keeps_the_right_slots(lib, hk, d, kind, budget, recent, sinks):
    from tensorfold_b200 import _lib, lane_evict

    layers, lens = 2, [0, 1, 100, 101, 700, 64, 350]
    table, k, v, mass, pos, gen = cache(budget, layers, lens, hk, d)
    if kind == "ties":
        mass = (mass * 4).round() / 4
    elif kind == "zeros":
        mass = torch.where(torch.rand(mass.shape, generator=gen) < 0.9, torch.where(torch.rand(mass.shape, generator=gen) < 0.5, 0.0, -0.0), mass)
    elif kind == "strange":
        for x in (math.nan, math.inf, -math.inf, -1.0, 1e-45):
            mass = torch.where(torch.rand(mass.shape, generator=gen) < 0.1, torch.tensor(x), mass)
    nxt = []
    for s, n in enumerate(lens):
        pg, pl = cells(table, s, n)
        text = torch.arange(n) + torch.where(torch.arange(n) < sinks, 0, 50)
        for layer in range(layers):
            for head in range(hk):
                pos[layer, pg, head, pl] = text[torch.randperm(n, generator=gen)].to(torch.int32)
        nxt.append(n + 50)
    want = [t.clone() for t in (k, v, mass, pos)]
    moved = torch.zeros((layers, len(lens), hk), dtype=torch.int32)
    for s, n in enumerate(lens):
        if n <= budget:
            continue
        pg, pl = cells(table, s, n)
        for layer in range(layers):
            for head in range(hk):
                holes, fills = select(mass[layer, pg, head, pl].tolist(), pos[layer, pg, head, pl].tolist(), n, budget, recent, sinks, nxt[s])
                assert len(holes) == len(fills)
                moved[layer, s, head] = len(holes)
                for t, src in zip(want, (k, v, mass, pos)):
                    t[layer, pg[holes], head, pl[holes]] = src[layer, pg[fills], head, pl[fills]]
    dev = [t.cuda() for t in (k, v, mass, pos)]
    got = lane_evict.evict(dev[0], dev[1], table.cuda(), i32(lens).cuda(), i32(nxt).cuda(), dev[2], dev[3], budget, recent=recent, sinks=sinks, max_context=max(lens))
    _lib.status(got.device).raise_if_set()
    assert torch.equal(got.cpu(), moved)
    for a, b, what in zip(dev, want, ("k", "v", "mass", "pos")):
        assert_same_bits(a.cpu(), b, what)


def test_evict_longer_than_shared_memory(lib):
    """More slots than a block's shared memory holds keys for."""

    from tensorfold_b200 import lane_evict

    n, budget = 60000, 20000
    table, k, v, mass, pos, gen = cache(1, 1, [n], 1, 128)
    pos.zero_()
    pg, pl = cells(table, 0, n)
    pos[0, pg, 0, pl] = torch.arange(n).to(torch.int32)
    order = torch.argsort(torch.where(torch.arange(n) >= n - 100, math.inf, mass[0, pg, 0, pl].double()), descending=True, stable=True)[:budget]
    kept = torch.zeros(n, dtype=torch.bool)
    kept[order] = True
    holes, fills = (~kept[:budget]).nonzero().flatten(), budget + kept[budget:].nonzero().flatten()
    want = k.clone()
    want[0, pg[holes], 0, pl[holes]] = k[0, pg[fills], 0, pl[fills]]
    dev = [t.cuda() for t in (k, v, mass, pos)]
    moved = lane_evict.evict(dev[0], dev[1], table.cuda(), i32([n]).cuda(), i32([n]).cuda(), dev[2], dev[3], budget, recent=100, max_context=n)
    assert int(moved) == len(holes)
    assert_same_bits(dev[0].cpu(), want)


def test_capture_and_reports(lib):
    from tensorfold_b200 import _lib, lane_evict

    lens, budget = [200, 90], 100
    table, k, v, mass, pos, _ = cache(4, 1, lens, 2, 128)
    pos.zero_().add_(5)
    base = [t.cuda() for t in (k, v, mass, pos)]
    eager = [t.clone() for t in base]
    t, l, x = table.cuda(), i32(lens).cuda(), i32([200, 90]).cuda()
    want = lane_evict.evict(eager[0], eager[1], t, l, x, eager[2], eager[3], budget, recent=10, max_context=200)
    work = [a.clone() for a in base]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moved = lane_evict.evict(work[0], work[1], t, l, x, work[2], work[3], budget, recent=10, max_context=200)
    for a, b in zip(work, base):
        a.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(moved, want)
    for a, b in zip(work, eager):
        assert_same_bits(a, b)
    status = _lib.status(t.device)
    status.raise_if_set()
    # a length above max_context, a page number that is none: reported
    lane_evict.evict(work[0], work[1], t, l, x, work[2], work[3], budget, recent=10, max_context=150)
    with pytest.raises(RuntimeError):
        status.raise_if_set()
    t[0, 3] = 10 ** 6
    lane_evict.evict(work[0], work[1], t, l, x, work[2], work[3], budget, recent=10, max_context=200)
    with pytest.raises(RuntimeError):
        status.raise_if_set()
    for kw in (dict(recent=99, sinks=2), dict(recent=-1), dict(recent=0, max_context=0)):
        with pytest.raises(ValueError):
            lane_evict.evict(work[0], work[1], t, l, x, work[2], work[3], budget, **{"max_context": 200, **kw})
    with pytest.raises(ValueError):
        lane_evict.evict(work[0], work[1], t, l, x, work[2][:, :1], work[3], budget, recent=0, max_context=200)
    with pytest.raises(ValueError):
        lane_evict.evict(work[0], work[1], t, l.long(), x, work[2], work[3], budget, recent=0, max_context=200)
