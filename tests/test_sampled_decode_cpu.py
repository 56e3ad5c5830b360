"""The round loop of ``decode.sampled_decode`` by itself, on the CPU: forward, verification and commit are stand-ins that note what they are given."""

from types import SimpleNamespace

import pytest
import torch

VOCAB = 64


@pytest.fixture
def loop(monkeypatch):
    """``loop.run(draft, count, seqs, ...)`` -> tokens; ``loop.calls``: the verifications' arguments; ``loop.commits``: what was committed."""

    from tensorfold_b200 import decode

    me = SimpleNamespace(calls=[], commits=[], keep=None, next=None, width=VOCAB)

    def tree_forward(w, tokens, widths, st):
        starts = [0]
        for x in widths:
            starts.append(starts[-1] + x)
        start = torch.tensor(starts, dtype=torch.int32)
        return torch.zeros((len(tokens), me.width), dtype=torch.bfloat16), SimpleNamespace(batch=SimpleNamespace(seq_start=start))

    def verify_drafts(logits, tokens, seq_start, uniforms, **kw):
        me.calls.append(SimpleNamespace(logits=logits, tokens=tokens, uniforms=uniforms, **kw))
        widths = (seq_start[1:] - seq_start[:-1]).tolist()
        keep = me.keep(widths) if me.keep else widths
        token = me.next(widths) if me.next else [7 if x else -1 for x in widths]
        return torch.tensor(keep, dtype=torch.int32), torch.tensor(token, dtype=torch.int32)

    monkeypatch.setattr(decode, "tree_forward", tree_forward)
    monkeypatch.setattr(decode, "verify_drafts", verify_drafts)
    monkeypatch.setattr(decode, "commit", lambda st, rec, keep: me.commits.append(list(keep)))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)

    def run(draft, count=6, seqs=1, **kw):
        w = SimpleNamespace(norm=torch.zeros(1), config=SimpleNamespace(vocab=VOCAB))
        return decode.sampled_decode(w, SimpleNamespace(n_seqs=seqs, position=lambda s: 3), [[1, 2, 3]] * seqs, [4] * seqs, count, draft=draft, **kw).tokens

    me.run = run
    return me


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.float64, torch.int32])
def test_drafters_logits_that_verification_would_round_are_refused(loop, dtype):
    """q is the softmax of the logits that the guesses were drawn from; rounded to bf16 they are another distribution's."""

    with pytest.raises(ValueError, match="bf16"):
        loop.run(lambda s, ctx, k: ([5] * k, torch.zeros((k, VOCAB), dtype=dtype)))
    assert not loop.commits


def test_drafters_logits_reach_verification_as_they_are(loop):
    theirs = torch.randn((8, VOCAB), generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    assert loop.run(lambda s, ctx, k: ([5] * k, theirs[:k]), seqs=2)[1] == [4] + [5] * 4 + [7]
    near = loop.calls[0].draft_logits
    assert near.dtype == torch.bfloat16 and torch.equal(near[1:5], theirs[:4]) and torch.equal(near[6:10], theirs[:4])


def test_random_numbers_have_64_bits(loop):
    """A vocabulary of 248320 has more borders than numbers of 24 bits tell apart evenly: 67 or 68 of them a token."""

    loop.run(lambda s, ctx, k: [5] * k, count=80, seqs=2, generator=torch.Generator().manual_seed(3))
    for call in loop.calls:
        assert call.uniforms.dtype == torch.float64 and call.uniforms.shape == (len(call.tokens), 2)
        assert bool(((call.uniforms >= 0) & (call.uniforms < 1)).all())
    drawn = torch.cat([c.uniforms for c in loop.calls]).flatten() * 2.0 ** 24
    assert float((drawn == drawn.floor()).double().mean()) < 0.01


def test_a_row_without_probabilities_ends_the_run(loop):
    """Verification answers -1 where every logit is -inf or NaN: no token, and nothing of that round is committed."""

    rounds = iter([[9, 9], [9, -1], [9, 9]])
    loop.next = lambda widths: next(rounds)
    loop.keep = lambda widths: [1] * len(widths)
    with pytest.raises(RuntimeError, match="sequence 1"):
        loop.run(lambda s, ctx, k: [5] * k, seqs=2, count=20)
    assert loop.commits == [[1, 1]]


def test_sequences_that_are_done_have_no_token(loop):
    """-1 is also what a sequence without rows gets."""

    loop.keep = lambda widths: [x if s == 0 else min(x, 1) for s, x in enumerate(widths)]
    tokens = loop.run(lambda s, ctx, k: [5] * k, seqs=2, count=6)
    assert [len(t) for t in tokens] == [6, 6] and any(0 in c for c in loop.commits)


def test_guesses_may_come_in_a_tuple(loop):
    """A pair is guesses and logits only where its second part can be logits."""

    for draft in (lambda s, ctx, k: (5, 6)[:k], lambda s, ctx, k: ((5, 6)[:k], None)):
        loop.calls.clear()
        assert loop.run(draft, count=4) == [[4, 5, 6, 7]]
        assert loop.calls[0].draft_logits is None


def test_padding_of_the_head_is_no_token(loop):
    """A head's rows come in eights (a vocabulary of 61 has 64 logits): what lies behind the vocabulary takes no part."""

    loop.width = VOCAB + 3
    theirs = torch.zeros((8, VOCAB), dtype=torch.bfloat16)
    assert len(loop.run(lambda s, ctx, k: ([5] * k, theirs[:k]))[0]) == 6
    assert len(loop.run(lambda s, ctx, k: [5] * k)[0]) == 6
    for call in loop.calls:
        assert call.logits.shape[1] == VOCAB and (call.draft_logits is None or call.draft_logits.shape == call.logits.shape)
