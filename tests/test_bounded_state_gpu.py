"""The bounded cache in use: rounds of attention, verification, commit, weights and eviction against a plain mirror, and models whose state has a
window or a budget."""

import math

import pytest
import torch

from oracle import lane_oracle as O
from tests.helpers import assert_same_bits

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")


def model(seed=31, layers=4, hk=2):
    from tensorfold_b200 import forward as F

    cfg = O.Config(hidden=256, intermediate=512, layers=layers, heads=4, kv_heads=hk, head_dim=128, vocab=512, k_heads=2, v_heads=4, dk=128, dv=128)
    return F.load_weights(O.random_model(cfg, seed=seed), "cuda")


def run(w, st, tokens, widths=None):
    from tensorfold_b200 import forward as F

    logits, rec = F.tree_forward(w, i32(tokens), widths or [len(tokens)], st)
    return logits, rec


def test_rounds_of_a_bounded_cache_against_a_mirror(lib):
    """Three sequences, eight rounds: window_attention(lse) -> verify_drafts -> kv_commit -> attention_mass -> evict, everything by `keep`
    as verification left it on the device; a mirror in 64 bits that holds each head's slots as lists. Its weights choose what goes, so a
    slot may differ only where the device's weights do not tell two apart by more than their error."""

    from tensorfold_b200 import _lib, lane_attention as LA, lane_evict, lane_window, speculative

    gen = torch.Generator().manual_seed(77)
    h, hk, d, v, budget, recent, sinks = 8, 2, 128, 300, 40, 8, 3
    g, seqs, scale = h // hk, 3, 128 ** -0.5
    kv = LA.PagedKV(1, seqs, 40, hk, d, 8, "cuda")
    kv.k.fill_(math.nan)                                       # stale rows are never read
    kv.v.fill_(math.nan)
    mass, pos = torch.full(kv.k.shape[:4], math.nan, device="cuda"), torch.full(kv.k.shape[:4], -9, dtype=torch.int32, device="cuda")
    lens, nxt = [0] * seqs, [0] * seqs
    mirror = [[dict(k=[], v=[], m=[], p=[]) for _ in range(hk)] for _ in range(seqs)]
    for rnd in range(8):
        widths = [[5, 1, 8], [8, 0, 8], [33, 8, 2], [8, 8, 8], [8, 30, 1], [2, 8, 8], [8, 8, 0], [8, 3, 8]][rnd]
        starts = [0]
        for x in widths:
            starts.append(starts[-1] + x)
        r = starts[-1]
        q = (2 * torch.randn((1, r, h, d), generator=gen)).to(BF)
        kn, vn = (torch.randn((1, r, hk, d), generator=gen).to(BF) for _ in range(2))
        for s in range(seqs):
            kv.reserve(s, max(lens[s] + widths[s], 1))
        kv.sync_table()
        lse, wide = torch.empty((1, r, h), device="cuda"), max(lens[s] + widths[s] for s in range(seqs))
        out = lane_window.window_attention(q[0].cuda(), kn[0].cuda(), vn[0].cuda(), kv.k[0], kv.v[0], kv.table, i32(lens), i32(starts), scale=scale,
                                           max_window=max(widths), max_context=wide, lse=lse[0])
        logits = (2 * torch.randn((r, v), generator=gen)).to(BF)
        keep, _ = speculative.verify_drafts(logits.cuda(), torch.randint(0, v, (r,), generator=gen).to(torch.int32).cuda(), i32(starts),
                                            (torch.rand((r, 2), generator=gen) * torch.tensor([2e-5, 1.0])).cuda())
        LA.kv_commit(kn.cuda(), vn.cuda(), kv, i32(lens), i32(starts), keep)
        row_pos = [nxt[s] + t for s in range(seqs) for t in range(widths[s])]
        lane_evict.attention_mass(q.cuda(), lse, kv.k, kv.table, i32(lens), i32(starts), keep, i32(row_pos), mass, pos, scale=scale, max_window=max(widths),
                                  max_context=wide)
        kept = keep.tolist()
        assert all(0 <= k <= w for k, w in zip(kept, widths)) and all(k >= 1 for k, w in zip(kept, widths) if w)
        for s in range(seqs):
            for head in range(hk):
                m = mirror[s][head]
                for t in range(widths[s]):
                    at = starts[s] + t
                    keys = torch.stack(m["k"] + [x.double() for x in kn[0, starts[s]:at + 1, head]])
                    vals = torch.stack(m["v"] + [x.double() for x in vn[0, starts[s]:at + 1, head]])
                    for a in range(head * g, head * g + g):
                        p = torch.softmax(keys @ q[0, at, a].double() * scale, 0)
                        want, size = p @ vals, p @ vals.abs()
                        # weights and results rounded to bf16, 2^-8 each; scores off by less than 2^-14
                        assert bool(((out[at, a].double().cpu() - want).abs() <= (2.0 ** -8 + 2.0 ** -12) * size + 2.0 ** -8 * want.abs()).all())
                for t in range(kept[s]):
                    m["k"].append(kn[0, starts[s] + t, head].double())
                    m["v"].append(vn[0, starts[s] + t, head].double())
                    m["m"].append(0.0)
                    m["p"].append(nxt[s] + t)
                for t in range(kept[s]):
                    n = lens[s] + t + 1
                    for a in range(head * g, head * g + g):
                        p = torch.softmax(torch.stack(m["k"][:n]) @ q[0, starts[s] + t, a].double() * scale, 0)
                        for j in range(n):
                            m["m"][j] += float(p[j])
            lens[s] += kept[s]
            nxt[s] += kept[s]
        moved = lane_evict.evict(kv.k, kv.v, kv.table, i32(lens), i32(nxt), mass, pos, budget, recent=recent, sinks=sinks, max_context=max(lens))
        for s in range(seqs):
            for head in range(hk):
                m, n = mirror[s][head], lens[s]
                if n > budget:
                    safe = [p < sinks or p >= nxt[s] - recent for p in m["p"]]
                    order = sorted(range(n), key=lambda j: (not safe[j], -m["m"][j], j))
                    stay = sorted(order[:budget])
                    holes, fills = [j for j in range(budget) if j not in stay], [j for j in stay if j >= budget]
                    assert int(moved[0, s, head]) == len(holes)
                    for name in m:
                        for a, b in zip(holes, fills):
                            m[name][a] = m[name][b]
                        del m[name][budget:]
                cells = [(int(kv.table_host[s, j // 16]), j % 16) for j in range(min(n, budget))]
                got_m = [float(mass[0, pg, head, pl]) for pg, pl in cells]
                got_p = [int(pos[0, pg, head, pl]) for pg, pl in cells]
                assert got_p == m["p"], (rnd, s, head)
                # each round's weights are off by less than 2^-12 of themselves
                assert all(abs(a - b) <= 2.0 ** -11 * b + 1e-7 for a, b in zip(got_m, m["m"]))
                for (pg, pl), kk, vv in zip(cells, m["k"], m["v"]):
                    assert torch.equal(kv.k[0, pg, head, pl].double().cpu(), kk) and torch.equal(kv.v[0, pg, head, pl].double().cpu(), vv)
            if lens[s] > budget:
                lens[s] = budget
                kv.shrink(s, budget)
    _lib.status(torch.device("cuda", 0)).raise_if_set()
    assert sorted(nxt)[1] > budget + 8                          # evictions took place


@pytest.mark.parametrize("bound", [dict(window=24, sinks=4), dict(window=1000), dict(budget=500)])
def test_window_rows_have_the_bits_of_serial_steps(lib, bound):
    from tensorfold_b200 import forward as F

    w = model()
    tokens = torch.randint(0, 512, (60,), generator=torch.Generator().manual_seed(3)).tolist()
    a, b = F.State(w, 1, 128, **bound), F.State(w, 1, 128, **bound)
    rows = []
    for t in tokens:
        logits, rec = run(w, b, [t])
        F.commit(b, rec, [1])
        rows.append(logits)
    got, at = [], 0
    for width in (13, 1, 8, 8, 16, 8, 6):
        logits, rec = run(w, a, tokens[at:at + width])
        F.commit(a, rec, [width])
        got.append(logits)
        at += width
    assert_same_bits(torch.cat(got), torch.cat(rows))


def test_a_wide_window_is_the_whole_cache(lib):
    """No key is out of sight yet: the bounded state's logits are the ordinary state's up to the roundings of two attention kernels, each
    within 4 % of the logits' range of the same 32-bit forward (the framework's bound for one layer in four)."""

    from tensorfold_b200 import forward as F

    w = model(5)
    tokens = torch.randint(0, 512, (90,), generator=torch.Generator().manual_seed(4)).tolist()
    plain, win, cut = F.State(w, 1, 128), F.State(w, 1, 128, window=200, sinks=4), F.State(w, 1, 128, budget=100, recent=10)
    want, _ = run(w, plain, tokens)
    for st in (win, cut):
        got, _ = run(w, st, tokens)
        assert float((got.float() - want.float()).abs().max()) <= 0.08 * float(want.float().abs().max())


def test_window_state_lives_in_few_pages_and_drafts_change_nothing(lib):
    from tensorfold_b200 import decode, forward as F

    w = model(9)
    prompts = [torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (150, 40)]
    results = []
    for kind in ("serial", "drafted"):
        st = F.State(w, 2, 400, window=48, sinks=5)                        # pages for the rows in sight and in flight, 450 positions or not
        assert st.kv.num_pages == 2 * (1 + 11 + 2)
        pending = decode.prefill(w, st, prompts, chunk=16)
        if kind == "serial":
            res = decode.serial_decode(w, st, pending, 120)
        else:
            res = decode.draft_decode(w, st, prompts, pending, 120, draft=lambda s, ctx, k: [(ctx[-1] + 1 + i * s) % 512 for i in range(k)])
        assert st.lens[0] >= 260 and len(st.kv.free) >= 28 - 2 * 9
        results.append(res.tokens)
    assert results[0] == results[1]


def test_budget_state_keeps_first_recent_and_heavy(lib):
    from tensorfold_b200 import _lib, decode, forward as F

    w = model(13)
    budget, recent, sinks = 70, 20, 4
    prompt = torch.randint(0, 512, (333,), generator=torch.Generator().manual_seed(8)).tolist()
    st = F.State(w, 1, 5000, budget=budget, recent=recent, sinks=sinks)
    assert st.kv.num_pages <= -(-(budget + 2 * 128 + 16) // 16)
    pending = decode.prefill(w, st, [prompt], chunk=100)
    assert st.position(0) == 333 and st.lens[0] <= budget + F.EVICT_SPARE and st.dropped[0] > 0
    res = decode.serial_decode(w, st, pending, 200)
    assert len(res.tokens[0]) == 200 and st.position(0) == 333 + 199 and st.lens[0] <= budget + F.EVICT_SPARE
    n = st.lens[0]
    cells = [(int(st.kv.table_host[0, j // 16]), j % 16) for j in range(n)]
    for head in range(2):
        at = [int(st.pos[0, pg, head, pl]) for pg, pl in cells]
        assert len(set(at)) == n and set(range(sinks)) <= set(at) and set(range(532 - recent, 532)) <= set(at) and max(at) == 531
        weight = torch.stack([st.mass[0, pg, head, pl] for pg, pl in cells])
        assert bool((weight >= 0).all()) and bool(weight.isfinite().all())
        # every row gave each of its head's two query heads' weights 1 in all; what left took its share along
        assert float(weight.sum()) <= 2 * 532 * (1 + 2.0 ** -10)
    _lib.status(st.seq_lens.device).raise_if_set()


def test_runner_with_a_bounded_state(lib):
    """The captured step gives the eager step's bits, also after pages have changed hands."""

    from tensorfold_b200 import forward as F
    from tensorfold_b200.runner import LaneRunner

    w = model(17)
    gen = torch.Generator().manual_seed(1)
    for bound in (dict(window=40, sinks=4), dict(budget=30, recent=8, sinks=2)):
        a, b = F.State(w, 2, 400, **bound), F.State(w, 2, 400, **bound)
        runner = LaneRunner(w, a, [8, 5], max_context=300)
        runner.refresh()
        runner.capture()
        for _ in range(30):
            tokens = torch.randint(0, 512, (13,), generator=gen).tolist()
            runner.step(tokens)
            logits, rec = run(w, b, tokens, [8, 5])
            assert_same_bits(runner.logits, logits)
            keep = torch.randint(1, 6, (2,), generator=gen).tolist()
            runner.commit(keep)
            F.commit(b, rec, keep)
            assert a.lens == b.lens and a.dropped == b.dropped


def test_snapshots_of_bounded_states(lib):
    from tensorfold_b200 import forward as F

    w = model(19)
    tokens = torch.randint(0, 512, (120,), generator=torch.Generator().manual_seed(2)).tolist()

    def advance(st, n):
        logits = None
        for at in range(0, n, 10):
            logits, rec = run(w, st, tokens[at:at + 10])
            F.commit(st, rec, [10])
        return logits

    st = F.State(w, 1, 400, budget=60, recent=8)
    advance(st, 50)
    snap = st.snapshot()
    first, _ = run(w, st, tokens[:8])
    mass = st.mass.clone()
    advance(st, 40)
    st.restore(snap)
    again, _ = run(w, st, tokens[:8])
    assert_same_bits(again, first)
    assert torch.equal(st.mass, mass)
    for _ in range(3):
        advance(st, 100)
    assert st.dropped[0] > 0
    with pytest.raises(ValueError):
        st.restore(snap)
    st = F.State(w, 1, 400, window=37)
    advance(st, 100)                                           # sees positions from 64 on: page 4, and at 110 positions from 74 on: still page 4
    snap = st.snapshot()
    advance(st, 10)
    st.restore(snap)
    advance(st, 60)
    with pytest.raises(ValueError):
        st.restore(snap)


def test_sampled_decode(lib):
    """At a temperature near zero every token is a largest logit, with and without a drafter's probabilities; a drafter that is the target itself
    is always kept; all rounds end with the tokens that were asked for."""

    from tensorfold_b200 import decode, forward as F

    w = model(23)
    prompts = [[1, 2, 3, 4, 1, 2, 3, 4, 1, 2], [7, 8, 9]]
    gen = torch.Generator(device="cuda").manual_seed(0)

    def drafter(s, ctx, k):
        logits = torch.randn((k, 512), generator=torch.Generator().manual_seed(len(ctx))).cuda().to(BF)
        return (logits.argmax(1).tolist(), logits) if s == 0 else [5] * k

    for draft in (None, drafter):
        st = F.State(w, 2, 200)
        pending = decode.prefill(w, st, prompts)
        res = decode.sampled_decode(w, st, prompts, pending, 30, temperature=1e-6, generator=gen, draft=draft)
        assert [len(t) for t in res.tokens] == [30, 30]
        check = F.State(w, 2, 200)
        decode.prefill(w, check, prompts)
        for i in range(29):
            logits, rec = run(w, check, [res.tokens[0][i], res.tokens[1][i]], [1, 1])
            for s in range(2):
                assert float(logits[s, res.tokens[s][i + 1]]) == float(logits[s].max())
            F.commit(check, rec, [1, 1])

    st = F.State(w, 1, 300)
    twin = F.State(w, 1, 300)
    pending = decode.prefill(w, st, prompts[:1])
    decode.prefill(w, twin, prompts[:1])
    seen = [0]

    def target(s, ctx, k):
        """The target's own distributions, drawn from: serial steps of a second state, taken back afterwards."""

        done = len(prompts[0]) + 0
        while twin.lens[0] < len(ctx) - 1:
            logits, rec = run(w, twin, [ctx[twin.lens[0]]])
            F.commit(twin, rec, [1])
        snap = twin.snapshot()
        guesses, rows, last = [], [], ctx[-1]
        for _ in range(k):
            logits, rec = run(w, twin, [last])
            F.commit(twin, rec, [1])
            last = int(torch.multinomial(torch.softmax(logits[0].float(), 0), 1, generator=gen))
            guesses.append(last)
            rows.append(logits)
        twin.restore(snap)
        seen[0] += k
        return (guesses, torch.cat(rows)) if k else []

    res = decode.sampled_decode(w, st, prompts[:1], pending, 60, generator=gen, draft=target, max_rows=6)
    # p = q to the bit: the draft is kept while u q < p, always
    assert res.accepted_drafts == res.drafted_rows == seen[0] and len(res.tokens[0]) == 60


def test_launches_are_counted(lib):
    from tensorfold_b200 import _lib, lane_window

    for seqs, launches in ((2, 1), (80, 2)):
        q, kn, pages = (torch.zeros(x, dtype=BF, device="cuda") for x in ((seqs, 8, 128), (seqs, 4, 128), (1, 4, 16, 128)))
        before = _lib.launch_count()
        lane_window.window_attention(q, kn, kn, pages, pages, i32([[0]] * seqs), i32([0] * seqs), i32(range(seqs + 1)), scale=1.0, max_window=1,
                                     max_context=16)
        assert _lib.launch_count() - before == launches


def test_what_drafters_return_is_checked(lib):
    from tensorfold_b200 import decode, forward as F

    w = model(3)
    for bad in ([512], [-1], ([5], torch.zeros((1, 511), device="cuda")), ([5, 6], torch.zeros((1, 512), device="cuda"))):
        st = F.State(w, 1, 64)
        pending = decode.prefill(w, st, [[1, 2, 3]])
        with pytest.raises(ValueError):
            decode.sampled_decode(w, st, [[1, 2, 3]], pending, 8, draft=lambda s, ctx, k: bad)


def test_engine_with_bounds(lib):
    """Two requests, the second an extension of the first, in far fewer pages than they have positions; a fresh start repeats the first."""

    from tensorfold_b200 import decode

    w = model(41)
    prompt = torch.randint(0, 512, (150,), generator=torch.Generator().manual_seed(6)).tolist()
    for bound in (dict(window=40, sinks=4), dict(budget=64, recent=16, sinks=4)):
        eng = decode.Engine(w, max_context=1000, **bound)
        first = eng.generate(prompt, 60)["tokens"]
        assert len(first) == 60
        assert len(eng.generate(prompt + first + [7], 300)["tokens"]) == 300
        assert eng.state.position(0) == len(prompt) + len(first) + 1 + 299 and eng.state.kv.num_pages < 25
        eng._reset()
        assert eng.generate(prompt, 60)["tokens"] == first


def test_bounds_are_checked(lib):
    from tensorfold_b200 import forward as F

    w = model(3)
    for bad in (dict(window=0), dict(window=5, budget=9), dict(budget=0), dict(budget=10, recent=8, sinks=3), dict(sinks=1), dict(recent=1), dict(window=9, sinks=-1)):
        with pytest.raises(ValueError):
            F.State(w, 1, 64, **bad)


def test_offsets_beyond_32_bits(lib):
    """Pages that lie more than 2^32 values into a cache: the bits of the same pages at its front."""

    from tensorfold_b200 import _lib, lane_evict, lane_window

    h, hk, d, n, w = 4, 1, 256, 90, 3
    gen = torch.Generator().manual_seed(12)
    count, used = (1 << 20) + 64, 6                            # 2^32 values of K and as many of V: 8.6 GB each
    rows, fill = (torch.randn((w, hk, d), generator=gen).to(BF).cuda() for _ in range(2)), torch.randn((2, used, hk, 16, d), generator=gen).to(BF).cuda()
    rows = list(rows)
    q = torch.randn((w, h, d), generator=gen).to(BF).cuda()
    results = []
    for first, total in ((0, used), (count - used, count)):
        k, v = torch.empty((1, total, hk, 16, d), dtype=BF, device="cuda"), torch.empty((1, total, hk, 16, d), dtype=BF, device="cuda")
        k[0, first:], v[0, first:] = fill[0], fill[1]
        mass, pos = torch.zeros((1, total, hk, 16), device="cuda"), torch.zeros((1, total, hk, 16), dtype=torch.int32, device="cuda")
        mass[0, first:] = torch.arange(used * 16, device="cuda").reshape(used, 1, 16).flip(0).float()
        pos[0, first:] = 50
        table, lens, start = i32([[first + i for i in range(used)]]), i32([n]), i32([0, w])
        lse = torch.empty((1, w, h), device="cuda")
        out = lane_window.window_attention(q, *rows, k[0], v[0], table, lens, start, scale=0.1, max_window=w, max_context=n + w, lse=lse[0])
        lane_evict.attention_mass(q[None], lse, k, table, i32([n - w]), start, i32([w]), i32([7, 8, 9]), mass, pos, scale=0.1, max_window=w, max_context=n)
        moved = lane_evict.evict(k, v, table, i32([n]), i32([1000]), mass, pos, 40, recent=0, sinks=8, max_context=n)
        results.append([t.clone() for t in (out, lse, mass[0, first:], pos[0, first:], k[0, first:], v[0, first:], moved)])
        del k, v
    for a, b in zip(*results):
        assert_same_bits(a, b)
    assert int(results[0][-1]) > 0
    _lib.status(torch.device("cuda", 0)).raise_if_set()
    torch.cuda.empty_cache()


def test_two_streams_at_once(lib):
    """Calls of every kind on two streams, with nothing shared: each gives what it gives alone."""

    from tensorfold_b200 import lane_evict, lane_window, speculative

    def rounds(seed, d):
        gen = torch.Generator().manual_seed(seed)
        h, hk, s, used = 8, 2, 6, 40
        k, v = (torch.randn((2, s * used, hk, 16, d), generator=gen).to(BF).cuda() for _ in range(2))
        mass, pos = torch.rand((2, s * used, hk, 16), generator=gen).cuda(), torch.arange(16).repeat(2, s * used, hk, 1).to(torch.int32).cuda()
        q, kn, vn = (torch.randn((4 * s, x, d), generator=gen).to(BF).cuda() for x in (h, hk, hk))
        logits, tokens = torch.randn((4 * s, 5000), generator=gen).to(BF).cuda(), torch.randint(0, 5000, (4 * s,), generator=gen).to(torch.int32).cuda()
        u = torch.rand((4 * s, 2), generator=gen).cuda()
        table, lens, start = torch.randperm(s * used, generator=gen).to(torch.int32).reshape(s, used).cuda(), i32([600, 5, 333, 70, 480, 17]), i32(range(0, 4 * s + 1, 4))
        row_pos = i32([0] * (4 * s))
        yield
        for _ in range(6):
            lse = torch.empty((2, 4 * s, h), device="cuda")
            outs = [lane_window.window_attention(q, kn, vn, k[i], v[i], table, lens, start, scale=0.08, max_window=4, max_context=640, lse=lse[i]) for i in range(2)]
            keep, token = speculative.verify_drafts(logits, tokens, start, u, draft_logits=logits.flip(0))
            lane_evict.attention_mass(torch.stack([q, q]), lse, k, table, lens, start, keep, row_pos, mass, pos, scale=0.08, max_window=4, max_context=640)
            moved = lane_evict.evict(k, v, table, lens, lens, mass, pos, 300, recent=10, sinks=2, max_context=640)
            yield
        yield [*outs, lse, keep, token, mass, pos, k, v, moved]

    def drive(together):
        streams = [torch.cuda.Stream() for _ in range(2)]
        runs = [rounds(5, 128), rounds(6, 256)]
        results = [None, None]
        for r in runs:
            next(r)
        torch.cuda.synchronize()
        for _ in range(7):
            for i, (st, r) in enumerate(zip(streams, runs)):
                with torch.cuda.stream(st):
                    results[i] = next(r)
                if not together:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        return results

    for one, two in zip(drive(False), drive(True)):
        for a, b in zip(one, two):
            assert_same_bits(a, b)
