"""What is timed of one verify round over a bounded K/V cache: its attention, the bookkeeping of which cached keys are used, the
eviction of those that are not, and the decision over the drafted tokens.

* ``window``: attention of verify rows to a paged cache within a sliding window, with a few first tokens that stay visible.
* ``mass``: the attention weight that every cached key has received, brought up to date after a commit, all layers at once.
* ``evict``: the cache of every layer and KV head cut back to a budget of slots by those weights.
* ``verify``: which drafted tokens are kept, and the next token, from the target's logits and given random numbers.

Where ``own`` is false the operators are computed in their plain form: elementary torch operations.
"""

import math
import random

import torch

own = False

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
PAGE = 16
NEVER = 1 << 30          # a window that no sequence reaches: all keys are visible


def _attend(name, seqs, width, ctx, window, sinks, heads=24, kv_heads=4, dim=256):
    """``width`` and ``ctx``: (smallest, largest) over the sequences; ``window`` 0: none."""

    return {"name": name, "kind": "window", "seqs": seqs, "width_lo": width[0], "width_hi": width[1], "ctx_lo": ctx[0], "ctx_hi": ctx[1],
            "window": window, "sinks": sinks, "heads": heads, "kv_heads": kv_heads, "dim": dim}


def _mass(name, layers, seqs, width, ctx, heads=24, kv_heads=4, dim=256):
    return {"name": name, "kind": "mass", "layers": layers, "seqs": seqs, "width_lo": width[0], "width_hi": width[1], "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "heads": heads, "kv_heads": kv_heads, "dim": dim}


def _evict(name, layers, seqs, ctx, budget, recent, sinks, kv_heads=4, dim=256):
    return {"name": name, "kind": "evict", "layers": layers, "seqs": seqs, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "budget": budget,
            "recent": recent, "sinks": sinks, "kv_heads": kv_heads, "dim": dim}


def _verify(name, seqs, width, vocab, drafter, temperature):
    return {"name": name, "kind": "verify", "seqs": seqs, "width_lo": width[0], "width_hi": width[1], "vocab": vocab, "drafter": drafter,
            "temperature": temperature}


def listed():
    return [
        # one user, no drafts: a serial token of a long conversation, one layer
        _attend("window_one_token", 1, (1, 1), (5000, 5000), 1024, 4),
        # one user with a drafter over the whole of a cache that eviction keeps bounded: no window, an uneven length
        _attend("window_whole_cache", 1, (8, 8), (4171, 4171), 0, 0),
        # a busy server: 16 users, ragged windows of drafts, contexts below and far above the window
        _attend("window_16_users", 16, (2, 8), (1500, 32768), 4096, 16),
        # a long prompt's rows in one call, on smaller heads, behind a committed prefix
        _attend("window_prompt", 2, (900, 2000), (333, 1500), 1024, 4, heads=16, kv_heads=2, dim=128),
        # one user's cache after a round that kept some of its rows, 16 attention layers
        _mass("mass_one_user", 16, 1, (4, 4), (4096, 4096)),
        # 16 users' caches, ragged, some of whom kept nothing but their first row; 4 layers
        _mass("mass_16_users", 4, 16, (1, 8), (2048, 8192)),
        # a cache a few rounds over its budget, 16 attention layers: what a user pays every few rounds
        _evict("evict_trickle", 16, 1, (4224, 4224), 4096, 512, 4),
        # long prompts cut back to the budget once they are processed, several users
        _evict("evict_prompts", 4, 4, (3000, 9000), 4096, 1024, 16),
        # one user whose drafts are copies of the context (no drafter's probabilities), the package's vocabulary
        _verify("verify_one_user", 1, (8, 8), 248320, False, 1.0),
        # a few users with a drafter, a small vocabulary of odd size
        _verify("verify_small_vocab", 3, (1, 5), 32003, True, 0.7),
        # 16 users x 8 rows with a drafter: a full step
        _verify("verify_16_users", 16, (8, 8), 248320, True, 0.8),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["window", "window", "window", "mass", "evict", "verify", "verify"])
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        heads, kv_heads, dim = rng.choice([(24, 4, 256), (16, 2, 128), (6, 1, 256), (16, 1, 256), (8, 8, 128), (32, 4, 128)])
        if kind == "window":
            what = rng.choice(["drafts", "drafts", "prompt"])
            lo, ctx = (rng.randint(1, 8), _log(rng, 40, 32768)) if what == "drafts" else (_log(rng, 20, 1000), _log(rng, 16, 4000))
            case = _attend("", _log(rng, 1, 24) if what == "drafts" else rng.randint(1, 3), (lo, rng.randint(lo, 8) if what == "drafts" else 2 * lo),
                           (max(1, ctx // 2), ctx), rng.choice([0, _log(rng, 60, 8192)]), rng.choice([0, 1, 4, 16, 70]), heads, kv_heads, dim)
        elif kind == "mass":
            lo, ctx = rng.randint(1, 8), _log(rng, 40, 16384)
            case = _mass("", rng.choice([1, 2, 5, 16]), _log(rng, 1, 24), (lo, rng.randint(lo, 8)), (max(1, ctx // 2), ctx), heads, kv_heads, dim)
        elif kind == "evict":
            budget = _log(rng, 50, 8192)
            case = _evict("", rng.choice([1, 2, 5, 16]), _log(rng, 1, 12), (budget // 2, _log(rng, budget + 1, 4 * budget)), budget,
                          _log(rng, 4, max(5, budget // 2)), rng.choice([0, 4, 16]), kv_heads, dim)
        else:
            lo = rng.randint(1, 8)
            case = _verify("", _log(rng, 1, 16), (lo, rng.randint(lo, 8)), _log(rng, 1000, 250000), rng.random() < 0.5, rng.choice([0.5, 0.8, 1.0, 1.3]))
        if _cost(case) <= most:
            del case["name"]
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def _layout(case):
    """Each sequence's window width, context and kept rows: a fixed function of the case (the same work for every seed)."""

    rng = random.Random(case["seqs"] * 1000 + case.get("width_hi", 0) + case.get("ctx_hi", 0))
    ctx = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])] if "ctx_lo" in case else None
    if "width_lo" not in case:
        return ctx, None, None
    widths = [rng.randint(case["width_lo"], case["width_hi"]) for _ in range(case["seqs"])]
    return ctx, widths, [rng.randint(1, w) for w in widths]


def _moved(case, n):
    """Slots that an eviction of a sequence of ``n`` slots is expected to move: the kept ones among those above the budget."""

    over, recent = n - case["budget"], case["recent"]
    if over <= 0:
        return 0
    share = (case["budget"] - recent) / (n - recent)
    return min(case["budget"], recent + (over - recent) * share if over > recent else over)


def work(case):
    kind = case["kind"]
    ctx, widths, kept = _layout(case)
    if kind == "verify":
        return {"bytes": sum(widths) * case["vocab"] * 2 * (2 if case["drafter"] else 1), "flops": 0}
    hk, d = case["kv_heads"], case["dim"]
    if kind == "window":
        window, sinks, h = case["window"] or NEVER, case["sinks"], case["heads"]
        seen = pairs = 0
        for n, w in zip(ctx, widths):
            first = max(0, n + 1 - window)                     # first key in the first row's window
            seen += min(sinks, first) + n + w - first
            at = [(min(window, p + 1), p + 1) for p in range(n, n + w)]
            pairs += sum(a + min(sinks, b - a) for a, b in at)
        rows = sum(widths)
        return {"bytes": seen * hk * d * 4 + rows * h * (d * 4 + 4), "flops": 4 * pairs * h * d}
    if kind == "mass":
        keys = sum(n + k for n, k in zip(ctx, kept))
        pairs = sum(k * n + k * (k + 1) // 2 for n, k in zip(ctx, kept))
        return {"bytes": case["layers"] * (keys * hk * (d * 2 + 8) + sum(kept) * case["heads"] * (d * 2 + 4)),
                "flops": 2 * case["layers"] * pairs * case["heads"] * d}
    over = [n for n in ctx if n > case["budget"]]
    return {"bytes": case["layers"] * hk * (sum(over) * 8 + sum(_moved(case, n) for n in over) * (d * 4 + 8) * 2) + 1024, "flops": 0}


def _i32(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def _table(lens, gen):
    """A page table whose pages are handed out in random order, as after a server has run for a while, and the number of pages."""

    need = [-(-n // PAGE) for n in lens]
    order = torch.randperm(sum(need), generator=gen, device="cuda").to(I32)
    table = torch.zeros((len(lens), max(need)), dtype=I32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, sum(need)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    ctx, widths, kept = _layout(case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(BF16)

    def pages(*shape):                       # large: filled in place
        return torch.empty(shape, dtype=BF16, device="cuda").normal_(generator=gen)

    st = dict(case)
    if widths is not None:
        rows, starts = sum(widths), [0]
        for w in widths:
            starts.append(starts[-1] + w)
        st.update(rows=rows, seq_start=_i32(starts), max_window=max(widths),
                  row_seq=torch.tensor([s for s, w in enumerate(widths) for _ in range(w)], device="cuda"),
                  row_idx=torch.tensor([t for w in widths for t in range(w)], device="cuda"))
    if kind == "verify":
        v = case["vocab"]
        # a language model's distribution: a few likely tokens above a long tail, the drafter's close to the target's
        logits = torch.randn((rows, v), generator=gen, device="cuda") * 2.0
        top = torch.randint(0, v, (rows, 12), generator=gen, device="cuda")
        logits.scatter_(1, top, 8.0 + 4.0 * torch.rand((rows, 12), generator=gen, device="cuda"))
        near = logits + 0.7 * torch.randn((rows, v), generator=gen, device="cuda")
        # row r + 1's input token is a draw of the drafter for the place that row r's logits predict
        drawn = (near / case["temperature"] - torch.empty((rows, v), device="cuda").exponential_(generator=gen).log()).argmax(1)
        st.update(tokens=drawn.roll(1).to(I32), logits=logits.to(BF16), uniforms=torch.rand((rows, 2), generator=gen, device="cuda"),
                  draft_logits=near.roll(1, 0).to(BF16) if case["drafter"] else None)
        return st
    hk, d = case["kv_heads"], case["dim"]
    lens = [n + w for n, w in zip(ctx, widths)] if widths is not None else ctx
    table, count = _table(lens, gen)
    st.update(table=table, lens=_i32(ctx), max_context=max(lens), scale=d ** -0.5)
    if kind == "window":
        h = case["heads"]
        st.update(q=normal(rows, h, d) * 2, k_new=normal(rows, hk, d), v_new=normal(rows, hk, d), k=pages(count, hk, PAGE, d), v=pages(count, hk, PAGE, d))
        return st
    layers = case["layers"]
    # where the slots of all sequences are: flat (page, place) numbers of the pool, and the (sequence, slot) pairs that exist
    every = torch.arange(table.shape[1] * PAGE, device="cuda")
    st["cell"] = table.long()[:, every // PAGE] * PAGE + every % PAGE
    st["k"] = pages(layers, count, hk, PAGE, d)
    heat = torch.empty((layers, count, hk, PAGE), dtype=F32, device="cuda").exponential_(generator=gen)
    if kind == "mass":
        h = case["heads"]
        after = [n + k for n, k in zip(ctx, kept)]
        st["q"] = normal(layers, rows, h, d) * 2
        # what the attention left: the rows' log-sum-exp over their keys, here near its expectation (scores of variance 4)
        st["lse"] = (torch.log(torch.tensor([float(n + t + 1) for n, w in zip(ctx, widths) for t in range(w)], device="cuda")).reshape(1, -1, 1) + 2.0
                     + 0.1 * torch.randn((layers, rows, h), generator=gen, device="cuda"))
        st.update(mass0=heat, mass=heat.clone(), pos=torch.zeros((layers, count, hk, PAGE), dtype=I32, device="cuda"), keep=_i32(kept),
                  row_pos=_i32([n + t for n, w in zip(ctx, widths) for t in range(w)]),
                  seq_of=torch.tensor([s for s, n in enumerate(after) for _ in range(n)], device="cuda"),
                  slot_of=torch.tensor([j for n in after for j in range(n)], device="cuda"))
        return st
    # a few keys hold most of the weight; a slot's position is its place in the text, the cache having been cut before or not
    st["v"] = pages(layers, count, hk, PAGE, d)
    st["mass0"] = heat ** 3
    pos = torch.zeros((layers, count * PAGE, hk), dtype=I32, device="cuda")
    nxt = []
    for s, n in enumerate(ctx):
        cut = n // 3
        nxt.append(n + cut)
        old = torch.arange(n, dtype=I32, device="cuda")
        old = torch.where(old < case["sinks"], old, old + cut)
        old[case["sinks"]:max(case["sinks"], n - 2 * case["recent"])] -= cut // 2
        if n > 2 * case["recent"] + case["sinks"]:            # earlier evictions have moved old slots about, not the latest ones
            mid = slice(case["sinks"], n - 2 * case["recent"])
            old[mid] = old[mid][torch.randperm(old[mid].numel(), generator=gen, device="cuda")]
        pos[:, st["cell"][s, :n]] = old.reshape(1, n, 1)
    st["pos0"] = pos.reshape(layers, count, PAGE, hk).transpose(2, 3).contiguous()
    st.update(mass=st["mass0"].clone(), pos=st["pos0"].clone(), next_pos=_i32(nxt))
    return st


def run(st):
    kind = st["kind"]
    if kind == "window":
        return _run_window(st)
    if kind == "verify":
        return _run_verify(st)
    st["mass"].copy_(st["mass0"])            # the weights are brought up to date in place: every pass starts from the same ones
    if kind == "mass":
        return _run_mass(st)
    st["pos"].copy_(st["pos0"])
    return _run_evict(st)


# ---- attention with a sliding window and sinks ---------------------------------------------------------------------------------
def _run_window(st):
    q, k_new, v_new = st["q"], st["k_new"], st["v_new"]
    rows, h, d = q.shape
    if own:
        from tensorfold_b200 import lane_window

        lse = torch.empty((rows, h), dtype=F32, device="cuda")
        out = lane_window.window_attention(q, k_new, v_new, st["k"], st["v"], st["table"], st["lens"], st["seq_start"], scale=st["scale"],
                                           window=st["window"] or None, sinks=st["sinks"], max_window=st["max_window"],
                                           max_context=st["max_context"], lse=lse)
        return {"out": out, "lse": lse}
    hk, window, sinks, wide = st["kv_heads"], st["window"] or NEVER, st["sinks"], st["max_window"]
    lens, start = st["lens"].long(), st["seq_start"].long()
    # the committed keys that any row of a sequence sees: its sinks, and what the first row's window holds
    first = (lens + 1 - window).clamp(min=0)
    near = torch.arange(min(window - 1, st["max_context"]), device="cuda") + torch.maximum(first, first.new_tensor(sinks)).reshape(-1, 1)
    at = torch.cat([torch.arange(sinks, device="cuda").expand(lens.numel(), sinks), near], 1)
    there = at < lens.reshape(-1, 1)
    clipped = torch.where(there, at, 0)
    page, place = st["table"].long().gather(1, clipped // PAGE), clipped % PAGE
    t = torch.arange(wide, device="cuda")
    width = start[1:] - start[:-1]
    row = torch.where(t < width.reshape(-1, 1), start[:-1].reshape(-1, 1) + t, 0)             # [S, W]
    keys = torch.cat([st["k"][page, :, place], k_new[row]], 1).float()                         # [S, keys, HK, D]
    vals = torch.cat([st["v"][page, :, place], v_new[row]], 1).float()
    where = torch.cat([at, lens.reshape(-1, 1) + t], 1)
    real = torch.cat([there, t < width.reshape(-1, 1)], 1)
    p = lens.reshape(-1, 1) + t                                                                # [S, W] the rows' places
    gap = p.unsqueeze(2) - where.unsqueeze(1)
    seen = real.unsqueeze(1) & (gap >= 0) & ((gap < window) | (where.unsqueeze(1) < sinks))
    qs = q[row].float().reshape(lens.numel(), wide, hk, h // hk, d)
    s = torch.einsum("swkgd,sjkd->skgwj", qs, keys) * st["scale"]
    s = s.masked_fill_(~seen.unsqueeze(1).unsqueeze(1), -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = (s - top).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.einsum("skgwj,sjkd->swkgd", e, vals) / total.squeeze(-1).permute(0, 3, 1, 2).unsqueeze(-1)
    lse = (total.log() + top).squeeze(-1).permute(0, 3, 1, 2).reshape(lens.numel(), wide, h)
    return {"out": o.reshape(lens.numel(), wide, h, d)[st["row_seq"], st["row_idx"]].to(BF16), "lse": lse[st["row_seq"], st["row_idx"]]}


# ---- accumulated attention weight ------------------------------------------------------------------------------------------------
def _run_mass(st):
    if own:
        from tensorfold_b200 import lane_evict

        lane_evict.attention_mass(st["q"], st["lse"], st["k"], st["table"], st["lens"], st["seq_start"], st["keep"], st["row_pos"], st["mass"],
                                  st["pos"], scale=st["scale"], max_window=st["max_window"], max_context=st["max_context"])
        return {"mass": st["mass"], "pos": st["pos"]}
    layers, rows, h, d = st["q"].shape
    hk, wide, n = st["kv_heads"], st["max_window"], st["max_context"]
    lens, start, keep = st["lens"].long(), st["seq_start"].long(), st["keep"].long()
    seqs = lens.numel()
    t, j = torch.arange(wide, device="cuda"), torch.arange(n, device="cuda")
    row = torch.where(t < keep.reshape(-1, 1), start[:-1].reshape(-1, 1) + t, 0)
    cell = st["cell"][:, :n]
    keys = st["k"][:, cell // PAGE, :, cell % PAGE].permute(2, 0, 1, 3, 4).float()             # [layers, S, keys, HK, D]
    qs = st["q"][:, row].float().reshape(layers, seqs, wide, hk, h // hk, d)
    s = torch.einsum("lswkgd,lsjkd->lskgwj", qs, keys) * st["scale"]
    s -= st["lse"][:, row].reshape(layers, seqs, wide, hk, h // hk).permute(0, 1, 3, 4, 2).unsqueeze(-1)
    seen = (t < keep.reshape(-1, 1)).unsqueeze(2) & (j <= (lens.reshape(-1, 1) + t).unsqueeze(2))
    added = s.exp_().masked_fill_(~seen.unsqueeze(1).unsqueeze(1), 0.0).sum((3, 4))            # [layers, S, HK, keys]
    sq, sl = st["seq_of"], st["slot_of"]
    c = cell[sq, sl]
    new = (sl >= lens[sq]).reshape(1, -1, 1)
    mass, pos = st["mass"], st["pos"]
    old = mass[:, c // PAGE, :, c % PAGE].permute(1, 0, 2)                                     # [layers, cells, HK]
    total = torch.where(new, 0.0, old) + added[:, sq, :, sl].permute(1, 0, 2)
    mass[:, c // PAGE, :, c % PAGE] = total.permute(1, 0, 2)
    was = pos[:, c // PAGE, :, c % PAGE].permute(1, 0, 2)
    place = st["row_pos"][(start[sq] + sl - lens[sq]).clamp(min=0, max=rows - 1)].reshape(1, -1, 1)
    pos[:, c // PAGE, :, c % PAGE] = torch.where(new, place, was).permute(1, 0, 2)
    return {"mass": mass, "pos": pos}


# ---- eviction ----------------------------------------------------------------------------------------------------------------------
def _run_evict(st):
    k, v, mass, pos, budget = st["k"], st["v"], st["mass"], st["pos"], st["budget"]
    if own:
        from tensorfold_b200 import lane_evict

        moved = lane_evict.evict(k, v, st["table"], st["lens"], st["next_pos"], mass, pos, budget, recent=st["recent"], sinks=st["sinks"],
                                 max_context=st["max_context"])
        return {"k": k, "v": v, "mass": mass, "pos": pos, "moved": moved}
    layers, hk, n = st["layers"], st["kv_heads"], st["max_context"]
    lens = st["lens"].long()
    seqs = lens.numel()
    cell = st["cell"][:, :n]
    j = torch.arange(n, device="cuda")
    heat = mass[:, cell // PAGE, :, cell % PAGE].permute(2, 0, 3, 1)                           # [layers, S, HK, slots]
    place = pos[:, cell // PAGE, :, cell % PAGE].permute(2, 0, 3, 1)
    held = (place < st["sinks"]) | (place >= (st["next_pos"].long() - st["recent"]).reshape(1, -1, 1, 1))
    there = (j < lens.reshape(-1, 1)).reshape(1, seqs, 1, n)
    rank = torch.where(there, torch.where(held, math.inf, heat), -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]                 # ties to the lower slot
    kept = torch.zeros((layers, seqs, hk, n), dtype=torch.bool, device="cuda").scatter_(-1, order, True) & there
    over = (lens > budget).reshape(1, seqs, 1, 1)
    below = j < budget
    hole, fill = ~kept & there & below & over, kept & ~below & over
    moved = fill.sum(-1)
    # the i-th kept slot above the budget goes into the i-th hole below it
    where_h, where_f = hole.nonzero(), fill.nonzero()
    to, frm = cell[where_h[:, 1], where_h[:, 3]], cell[where_f[:, 1], where_f[:, 3]]
    la, hd = where_h[:, 0], where_h[:, 2]
    for x in (k, v, mass, pos):
        x[la, to // PAGE, hd, to % PAGE] = x[la, frm // PAGE, hd, frm % PAGE]
    return {"k": k, "v": v, "mass": mass, "pos": pos, "moved": moved.to(I32)}


# ---- verification of drafted tokens ------------------------------------------------------------------------------------------------
def _run_verify(st):
    logits, near, tokens, u, temp = st["logits"], st["draft_logits"], st["tokens"], st["uniforms"], st["temperature"]
    if own:
        from tensorfold_b200 import speculative

        keep, token = speculative.verify_drafts(logits, tokens, st["seq_start"], u, temperature=temp, draft_logits=near, max_window=st["max_window"])
        return {"keep": keep, "token": token}
    start, wide = st["seq_start"].long(), st["max_window"]
    width = start[1:] - start[:-1]
    rows = logits.shape[0]
    # the normalisers in 64 bits: an acceptance is a comparison, and a draw is a place among 250000 borders
    x = logits.double() / temp
    lse = torch.logsumexp(x, 1)
    after = torch.arange(1, rows + 1, device="cuda").clamp(max=rows - 1)                       # the row whose input is the next draft
    drafted = tokens.long()[after].reshape(-1, 1)
    p_at = (x.gather(1, drafted).squeeze(1) - lse).exp()
    if near is None:
        q_at = torch.ones_like(p_at)
    else:
        y = near.double() / temp
        lse_q = torch.logsumexp(y, 1)
        q_at = (y[after].gather(1, drafted).squeeze(1) - lse_q[after]).exp()
    taken = u[:, 0].double() * q_at < p_at
    t = torch.arange(wide, device="cuda")
    row = torch.where(t < width.reshape(-1, 1), start[:-1].reshape(-1, 1) + t, 0)
    ok = taken[row] & (t < (width - 1).reshape(-1, 1))
    keep = ok.long().cumprod(1).sum(1) + 1
    at = start[:-1] + keep - 1                                                                 # the row that the next token comes from
    w = (x[at] - lse[at].reshape(-1, 1)).exp()
    full = (keep == width).reshape(-1, 1)
    if near is None:
        rest = w.scatter(1, drafted[at], 0.0)
    else:
        rest = (w - (y[after[at]] - lse_q[after[at]].reshape(-1, 1)).exp()).clamp(min=0.0)
    cdf = torch.where(full, w, rest).cumsum(1)
    token = (cdf <= u[at, 1].double().reshape(-1, 1) * cdf[:, -1:]).sum(1)
    return {"keep": keep.to(I32), "token": token.to(I32)}


# ---- the definitions in 64 bits, one sequence and head at a time ---------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"window": _exact_window, "mass": _exact_mass, "evict": _exact_evict, "verify": _exact_verify}[case["kind"]](case, st)


def _slots(pages, table_row, head, n):
    """Keys or values of a sequence's first n slots, [n, D] in 64 bits."""

    used = table_row[:-(-n // PAGE)].long()
    return pages[used, head].reshape(-1, pages.shape[-1])[:n].double()


def _exact_window(case, st):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    g = h // hk
    ctx, widths, _ = _layout(case)
    out = torch.empty((st["rows"], h, d), dtype=F64, device="cuda")
    lse = torch.empty((st["rows"], h), dtype=F64, device="cuda")
    r0 = 0
    for s, (n, w) in enumerate(zip(ctx, widths)):
        for head in range(hk):
            keys = torch.cat([_slots(st["k"], st["table"][s], head, n), st["k_new"][r0:r0 + w, head].double()])
            vals = torch.cat([_slots(st["v"], st["table"][s], head, n), st["v_new"][r0:r0 + w, head].double()])
            i, j = torch.arange(n, n + w, device="cuda").unsqueeze(1), torch.arange(n + w, device="cuda").unsqueeze(0)
            hidden = (j > i) | ((j <= i - (case["window"] or NEVER)) & (j >= case["sinks"]))
            for a in range(head * g, head * g + g):
                score = (st["q"][r0:r0 + w, a].double() @ keys.T * st["scale"]).masked_fill(hidden, -math.inf)
                lse[r0:r0 + w, a] = torch.logsumexp(score, 1)
                out[r0:r0 + w, a] = torch.softmax(score, 1) @ vals
        r0 += w
    return {"out": out, "lse": lse}


def _exact_mass(case, st):
    g = case["heads"] // case["kv_heads"]
    ctx, widths, kept = _layout(case)
    mass = st["mass0"].double()
    for layer in range(case["layers"]):
        r0 = 0
        for s, (n, w, m) in enumerate(zip(ctx, widths, kept)):
            slot = torch.arange(n + m, device="cuda")
            page = st["table"][s].long()[slot // PAGE]
            late = slot.unsqueeze(0) > torch.arange(n, n + m, device="cuda").unsqueeze(1)
            for head in range(case["kv_heads"]):
                keys = _slots(st["k"][layer], st["table"][s], head, n + m)
                total = mass[layer, page, head, slot % PAGE]
                total[n:] = 0.0
                for a in range(head * g, head * g + g):
                    score = st["q"][layer, r0:r0 + m, a].double() @ keys.T * st["scale"] - st["lse"][layer, r0:r0 + m, a].double().unsqueeze(1)
                    total += score.exp().masked_fill(late, 0.0).sum(0)
                mass[layer, page, head, slot % PAGE] = total
            r0 += w
    return {"mass": mass, "pos": None}


def _exact_evict(case, st):
    """The weights that stay, each head's slots ranked by themselves; what is moved is not computed."""

    ctx, _, _ = _layout(case)
    mass = st["mass0"].double()
    budget = case["budget"]
    for layer in range(case["layers"]):
        for s, n in enumerate(ctx):
            if n <= budget:
                continue
            slot = torch.arange(n, device="cuda")
            page = st["table"][s].long()[slot // PAGE]
            for head in range(case["kv_heads"]):
                heat, place = mass[layer, page, head, slot % PAGE], st["pos0"][layer, page, head, slot % PAGE].long()
                safe = (place < case["sinks"]) | (place + case["recent"] >= int(st["next_pos"][s]))
                best = torch.sort(torch.where(safe, math.inf, heat), descending=True, stable=True).indices[:budget]
                stays = torch.zeros(n, dtype=torch.bool, device="cuda")
                stays[best] = True
                holes, movers = slot[:budget][~stays[:budget]], slot[budget:][stays[budget:]]
                heat[holes] = heat[movers]
                mass[layer, page, head, slot % PAGE] = heat
    return {"k": None, "v": None, "mass": mass, "pos": None, "moved": None}


def _exact_verify(case, st):
    widths = _layout(case)[1]
    temp, tokens = case["temperature"], st["tokens"].tolist()
    keep, chosen, r0 = [], [], 0
    for w in widths:
        t = 0
        while True:
            p = torch.softmax(st["logits"][r0 + t].double() / temp, 0)
            if t + 1 == w:
                break
            x = tokens[r0 + t + 1]
            if st["draft_logits"] is None:
                q = torch.zeros_like(p)
                q[x] = 1.0
            else:
                q = torch.softmax(st["draft_logits"][r0 + t + 1].double() / temp, 0)
            if not float(st["uniforms"][r0 + t, 0]) * float(q[x]) < float(p[x]):
                p = torch.relu(p - q)
                break
            t += 1
        c = torch.cumsum(p, 0)
        keep.append(t + 1)
        chosen.append(int(torch.searchsorted(c, c[-1] * st["uniforms"][r0 + t, 1].double(), right=True)))
        r0 += w
    return {"keep": torch.tensor(keep, dtype=I32), "token": torch.tensor(chosen, dtype=I32)}
