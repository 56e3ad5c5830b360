"""``decode.sampled_decode`` on a model: its tokens' distribution, and logits that are none."""

import math

import pytest
import torch

from oracle import lane_oracle as O

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")


def model(seed, vocab=512):
    from tensorfold_b200 import forward as F

    cfg = O.Config(hidden=256, intermediate=512, layers=4, heads=4, kv_heads=2, head_dim=128, vocab=vocab, k_heads=2, v_heads=4, dk=128, dv=128)
    return F.load_weights(O.random_model(cfg, seed=seed), "cuda")


@pytest.mark.parametrize("kind", ["probabilities", "certain"])
def test_tokens_follow_the_target(lib, kind):
    """64 sequences with one text, many times over: the token behind it has the target's distribution, whatever the drafter proposes."""

    from tensorfold_b200 import decode, forward as F

    w, seqs, times, temp = model(5), 64, 120, 0.5
    prompt = [3, 1, 4, 1, 5, 9, 2, 6]
    st = F.State(w, seqs, 64)
    pending = decode.prefill(w, st, [prompt] * seqs, chunk=2)
    assert len(set(pending)) == 1
    snap = st.snapshot()
    logits, _ = F.tree_forward(w, i32(pending), [1] * seqs, st)
    p = torch.softmax(logits[0].double().cpu() / temp, 0)
    cpu, gen = torch.Generator().manual_seed(1), torch.Generator(device="cuda").manual_seed(2)
    near = (logits[0].float().cpu() + 1.5 * torch.randn(512, generator=cpu)).to(BF)
    q = torch.softmax(near.double() / 0.7, 0)
    counts = torch.zeros(512, dtype=torch.float64)

    def draft(s, ctx, k):
        if kind == "certain":
            return [int(p.argmax())] * min(k, 1)
        return torch.multinomial(q, 1, generator=cpu).tolist()[:k], near.unsqueeze(0).cuda()

    kept = 0
    for _ in range(times):
        st.restore(snap)
        res = decode.sampled_decode(w, st, [prompt] * seqs, pending, 3, temperature=temp, draft_temperature=0.7, generator=gen, draft=draft)
        counts += torch.bincount(torch.tensor([t[1] for t in res.tokens]), minlength=512).double()
        kept += res.accepted_drafts
    total = seqs * times
    assert 0 < kept
    # five standard deviations of a count of independent draws, for the tokens of which there are many and for the others together
    many = p * total >= 50
    share = torch.cat([p[many], p[~many].sum().reshape(1)])
    got = torch.cat([counts[many], counts[~many].sum().reshape(1)])
    assert int(many.sum()) >= 5
    assert bool(((got / total - share).abs() <= 5 * (share * (1 - share) / total).sqrt() + 1e-9).all()), (got / total - share)


def test_logits_that_are_none_end_the_run(lib):
    from tensorfold_b200 import decode, forward as F

    w = model(7)
    st = F.State(w, 2, 64)
    pending = decode.prefill(w, st, [[1, 2, 3], [4, 5]])
    w.norm.fill_(math.nan)
    with pytest.raises(RuntimeError, match="sequence 0"):
        decode.sampled_decode(w, st, [[1, 2, 3], [4, 5]], pending, 8)
    assert st.lens == [3, 2]


def test_a_vocabulary_that_is_no_multiple_of_eight(lib):
    """The head is padded with rows of zeros, whose logits are 0: above many a token's."""

    from tensorfold_b200 import decode, forward as F

    w = model(9, vocab=509)
    prompts = [[1, 2, 3], [4, 5]]
    st = F.State(w, 2, 300)
    pending = [7, 8]
    decode.prefill(w, st, prompts)
    gen = torch.Generator(device="cuda").manual_seed(1)
    near = torch.zeros((8, 509), dtype=BF, device="cuda")
    res = decode.sampled_decode(w, st, prompts, pending, 120, temperature=50.0, generator=gen, draft=lambda s, ctx, k: ([len(ctx) % 509] * k, near[:k]) if s else [5] * k)
    assert [len(t) for t in res.tokens] == [120, 120] and max(max(t) for t in res.tokens) < 509
