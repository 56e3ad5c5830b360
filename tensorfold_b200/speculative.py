"""Verification of drafted tokens against the target's probabilities, from given random numbers.

Beside ``exact_sampling.sample_rows`` with ``forward.accept_path``, where a draft is kept if it equals the token that the position's key
draws: here a draft is kept with probability min(1, p / q), and what replaces the first refused one is drawn from max(p - q, 0), so
that the tokens are distributed as the target's own whatever the drafter proposes, and a drafter that is close to the target is
kept more often than two separate draws agree. The reference has no counterpart.
"""

from __future__ import annotations

import torch

from . import _lib

def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, seq_start: torch.Tensor, uniforms: torch.Tensor, *, temperature: float = 1.0,
                  draft_logits: torch.Tensor | None = None, draft_temperature: float | None = None, max_window: int | None = None,
                  scratch: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(keep, next) int32 (S,) on the device: how many rows of each window are kept, and the token after the last of them.

    logits (R, V) bf16: the target's, of every window row; tokens (R,) int32: the rows' input tokens (a window's first is decided, the
    others are drafts); seq_start (S+1,) int32; uniforms (R, 2) float32 or float64 in [0, 1): row t's decide over the draft behind it and
    draw the token after it. With p = softmax(logits[t] / temperature) and q = softmax(draft_logits[t+1] / draft_temperature) the
    draft x = tokens[t+1] is kept while uniforms[t, 0] * q(x) < p(x). ``draft_logits`` (R, V) bf16: row t+1 holds what its token was
    drawn from (a window's first row is not read); None: the drafts are certain (copies of the context), q is all on x. The next
    token is the first in vocabulary order whose cumulative weight exceeds uniforms[t, 1] of the total, t the last kept row: of
    max(p - q, 0) if the draft behind it was refused, of p if the window was kept whole. Full distributions: no top-k or top-p.
    Temperatures in 1e-6..1e6 (greedy decoding: ``sample_rows`` and ``accept_path``).
    A sequence without rows gives (0, -1); a row without any probability keeps no draft and gives -1. ``max_window`` (the longest window) is not
    needed and changes nothing. ``keep`` is what ``kv_commit`` and ``lane_evict.attention_mass`` take.
    """

    if max_window is not None and max_window < 1:
        raise ValueError("verify_drafts: max_window must be positive")
    return _lib.host().verify_drafts(logits, tokens, seq_start, uniforms, temperature, draft_logits, draft_temperature, scratch)


__all__ = ["verify_drafts"]
