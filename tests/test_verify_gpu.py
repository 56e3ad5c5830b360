"""Verification of drafts: against the definition in 64 bits, at its borders, and that the tokens follow the target's distribution."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
i32 = lambda x: torch.tensor(x, dtype=torch.int32)


def tame(x):
    return torch.where(x.isnan(), -math.inf, x.double().clamp(max=float(torch.finfo(BF).max)))


def probs(row, temp):
    x = tame(row)
    if not bool((x > -math.inf).any()):
        return torch.full_like(x, math.nan)
    return torch.softmax(x / temp, 0)


def plain(logits, tokens, starts, u, temp, near, near_t):
    keep, nxt = [], []
    v = logits.shape[1]
    for r0, r1 in zip(starts, starts[1:]):
        if r0 == r1:
            keep.append(0)
            nxt.append(-1)
            continue
        t = r0
        while True:
            p = probs(logits[t], temp)
            if t == r1 - 1:
                w = p
                break
            x = int(tokens[t + 1])
            inside = 0 <= x < v
            q = probs(near[t + 1], near_t) if near is not None else torch.zeros_like(p)
            if near is None and inside:
                q[x] = 1.0
            if not (inside and float(u[t, 0]) * float(q[x]) < float(p[x])):
                w = (p - torch.where(q.isnan(), 0.0, q)).clamp(min=0.0)
                if not bool((w > 0).any()):
                    w = p
                break
            t += 1
        keep.append(t - r0 + 1)
        if bool(w.isnan().any()):
            nxt.append(-1)
            continue
        c = w.cumsum(0)
        nxt.append(int((c <= c[-1] * float(u[t, 1])).sum()))
    return keep, nxt


def case(seed, widths, v, sharp=3.0, extra=0):
    gen = torch.Generator().manual_seed(seed)
    starts = [0]
    for w in widths:
        starts.append(starts[-1] + w)
    r = starts[-1] + extra
    logits = (sharp * torch.randn((r, v), generator=gen)).to(BF)
    near = (logits.float() + torch.randn((r, v), generator=gen)).roll(1, 0).to(BF)
    tokens = torch.multinomial(torch.softmax(near.float() * 1.5, 1), 1, generator=gen).flatten().to(torch.int32)
    return logits, near, tokens, starts, torch.rand((r, 2), generator=gen)


def run(logits, tokens, starts, u, temp, near=None, near_t=None, **kw):
    from tensorfold_b200 import speculative

    keep, nxt = speculative.verify_drafts(logits.cuda(), tokens.cuda(), i32(starts).cuda(), u.cuda(), temperature=temp,
                                          draft_logits=None if near is None else near.cuda(), draft_temperature=near_t, **kw)
    assert keep.dtype == nxt.dtype == torch.int32
    return keep.tolist(), nxt.tolist()


@pytest.mark.parametrize("v", [1, 2, 7, 255, 1000, 8191, 8193, 32003, 70001])
@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("temp", [0.3, 1.0, 2.5])
def test_against_64_bits(lib, v, drafter, temp):
    logits, near, tokens, starts, u = case(v, [1, 4, 0, 8, 2, 3], v, extra=2)
    near = near if drafter else None
    for dtype in (torch.float32, torch.float64):
        assert run(logits, tokens, starts, u.to(dtype), temp, near, 0.8) == plain(logits, tokens, starts, u.to(dtype), temp, near, 0.8)


def test_many_rows_and_strides(lib):
    """More rows than a warp or a block has lanes, rows off a 16-byte boundary, rows that lie apart."""

    logits, near, tokens, starts, u = case(3, [100, 1, 60], 1001, sharp=1.0)
    near = near.clone()
    near[1:] = logits[:-1]                                   # the drafter is the target: nearly all is kept
    wide = torch.full((161, 1003), 9.0, dtype=BF)
    wide[:, 1:1002] = logits
    view = wide.cuda()[:, 1:1002]
    from tensorfold_b200 import speculative

    got = speculative.verify_drafts(view, tokens.cuda(), i32(starts).cuda(), u.cuda(), draft_logits=near.cuda(), max_window=100)
    want = plain(logits, tokens, starts, u, 1.0, near, 1.0)
    assert (got[0].tolist(), got[1].tolist()) == want
    assert want[0] == [100, 1, 60]


def test_borders(lib):
    v = 1000
    logits, near, tokens, starts, u = case(5, [3] * 8, v)
    u[:, 0] = 0.0                                            # everything with any probability is kept
    assert run(logits, tokens, starts, u, 1.0) == plain(logits, tokens, starts, u, 1.0, None, 1.0)
    u[:, 1] = 0.0                                            # the first token with any weight
    logits[:, :17] = -math.inf
    assert run(logits, tokens, starts, u, 1.0)[1] == plain(logits, tokens, starts, u, 1.0, None, 1.0)[1]
    u[:, 1] = 1 - 2.0 ** -24                                 # the last one
    logits[:, -9:] = -math.inf
    got = run(logits, tokens, starts, u, 1.0)
    assert got == plain(logits, tokens, starts, u, 1.0, None, 1.0) and all(t < v - 9 for t in got[1])
    u[:, 0] = 1 - 2.0 ** -24                                 # certain drafts are kept with probability p only
    assert run(logits, tokens, starts, u, 1.0)[0] == plain(logits, tokens, starts, u, 1.0, None, 1.0)[0]


def test_strange_logits_and_drafts(lib):
    v = 500
    logits, near, tokens, starts, u = case(6, [3] * 10, v)
    logits[0, 5] = math.inf                                  # all of it on one token, on two, on none
    logits[3, 5] = logits[3, 400] = math.inf
    logits[6] = -math.inf
    logits[9] = math.nan
    logits[12, ::2] = math.nan
    logits[15] = 0.0
    near[19] = -math.inf                                     # the drafter says nothing
    near[22, 3] = math.inf
    tokens[25], tokens[28] = -1, v                           # drafts outside the vocabulary
    for d in (None, near):
        got = run(logits, tokens, starts, u, 0.9, d, 0.9)
        assert got == plain(logits, tokens, starts, u, 0.9, d, 0.9)
        assert got[0][2:4] == [1, 1] and got[1][2:4] == [-1, -1]


def test_only_the_draft_has_any_probability(lib):
    """p is all on the draft: it is kept whatever the number; a refused draft that was all of p leaves p itself."""

    v = 64
    logits = torch.full((2, v), -math.inf).to(BF)
    logits[:, 7] = 1.0
    u = torch.tensor([[0.999999, 0.5], [0.5, 0.5]])
    assert run(logits, i32([3, 7]), [0, 2], u, 1.0) == ([2], [7])
    assert run(logits, i32([3, 8]), [0, 2], u, 1.0) == ([1], [7])
    near = logits.clone()
    assert run(logits, i32([3, 7]), [0, 2], torch.tensor([[1.0, 0.5], [0.5, 0.5]]), 1.0, near) == ([1], [7])     # q = p, refused by a number that is none


def test_tokens_follow_the_target(lib):
    """Whatever the drafter proposes, the token after the first row is the target's: 200000 windows of one draft over 6 tokens."""

    from tensorfold_b200 import speculative

    n, v = 16000, 6
    gen = torch.Generator(device="cuda").manual_seed(0)
    target = torch.tensor([1.0, 0.2, -1.0, 0.5, -3.0, 0.0]).to(BF)
    draft = torch.tensor([-1.0, 1.0, 0.3, 0.5, 0.0, -8.0]).to(BF)
    p, q = torch.softmax(target.double(), 0), torch.softmax(draft.double(), 0)
    counts, kept = torch.zeros(v, dtype=torch.float64), 0
    rounds = 8
    for _ in range(rounds):
        tokens = torch.multinomial(q.cuda().expand(2 * n, v).float(), 1, generator=gen).flatten().to(torch.int32)
        u = torch.rand((2 * n, 2), generator=gen, device="cuda", dtype=torch.float64)
        keep, nxt = speculative.verify_drafts(target.cuda().expand(2 * n, v).contiguous(), tokens, torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda"), u,
                                              draft_logits=draft.cuda().expand(2 * n, v).contiguous())
        first = torch.where(keep == 2, tokens[1::2], nxt).long()
        counts += torch.bincount(first, minlength=v).double().cpu()
        kept += int((keep == 2).sum())
    total = n * rounds
    # five standard deviations of a count over independent windows
    assert bool(((counts / total - p).abs() <= 5 * (p * (1 - p) / total).sqrt()).all()), counts / total - p
    rate = float(torch.minimum(p, q).sum())
    assert abs(kept / total - rate) <= 5 * math.sqrt(rate * (1 - rate) / total)


def test_sequences_that_are_not_among_the_rows(lib):
    """seq_start lies on the device, where no check of arguments sees it: such a sequence has no rows, the others are as ever."""

    from tensorfold_b200 import speculative

    logits, near, tokens, starts, u = case(9, [4, 2], 3001)
    dev = [logits.cuda(), tokens.cuda(), None, u.cuda()]
    right = plain(logits, tokens, starts, u, 1.0, near, 1.0)
    for bad, which in (([0, 4, 99], 0), ([-3, 4, 6], 1), ([0, 4, 2 ** 31 - 1], 0), ([-2 ** 31, 4, 6], 1)):
        dev[2] = i32(bad).cuda()
        keep, nxt = speculative.verify_drafts(*dev, draft_logits=near.cuda())
        torch.cuda.synchronize()
        assert keep.tolist()[which] == right[0][which] and nxt.tolist()[which] == right[1][which]
        assert keep.tolist()[1 - which] == 0 and nxt.tolist()[1 - which] == -1


def test_capture_and_refusals(lib):
    from tensorfold_b200 import speculative

    logits, near, tokens, starts, u = case(8, [4, 2], 3001)
    dev = [logits.cuda(), tokens.cuda(), i32(starts).cuda(), u.cuda()]
    drafter = near.cuda()
    speculative.verify_drafts(*dev, draft_logits=drafter)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep, nxt = speculative.verify_drafts(*dev, draft_logits=drafter)
    graph.replay()
    torch.cuda.synchronize()
    assert (keep.tolist(), nxt.tolist()) == plain(logits, tokens, starts, u, 1.0, near, 1.0)
    for kw in (dict(temperature=0.0), dict(temperature=math.inf), dict(temperature=math.nan), dict(draft_logits=near.cuda()[:, :9]), dict(draft_temperature=-1.0),
               dict(max_window=0), dict(scratch=torch.empty(8, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(ValueError):
            speculative.verify_drafts(*dev, **kw)
    for i, bad in ((0, dev[0].float()), (1, dev[1].long()), (1, dev[1][:3]), (2, dev[2].long()), (3, dev[3].half()), (3, dev[3][:, :1]), (2, dev[2].cpu()), (0, logits)):
        with pytest.raises(ValueError):
            speculative.verify_drafts(*[bad if j == i else t for j, t in enumerate(dev)])
