"""Verification of drafted tokens against the target's probabilities, from given random numbers.

Beside ``exact_sampling.sample_rows`` with ``forward.accept_path``, where a draft is kept if it equals the token that the position's key
draws: here a draft is kept with probability min(1, p / q), and what replaces the first refused one is drawn from max(p - q, 0), so
that the tokens are distributed as the target's own whatever the drafter proposes, and a drafter that is close to the target is
kept more often than two separate draws agree. The reference has no counterpart.
"""

from __future__ import annotations

import torch

from . import _lib

MAX_VOCAB = 1 << 20


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    if x.dim() != 2 or x.dtype != torch.bfloat16 or x.shape[0] < 1 or not 1 <= x.shape[1] <= MAX_VOCAB:
        raise ValueError(f"verify_drafts: {what} must be bf16 rows of 1..{MAX_VOCAB} logits")
    return x if x.stride(1) == 1 and x.stride(0) >= x.shape[1] else x.contiguous()


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
    A sequence without rows gives (0, -1); a row without any probability keeps no draft and gives -1. ``max_window`` only has to be at
    least the longest window and may be left out. ``keep`` is what ``kv_commit`` and ``lane_evict.attention_mass`` take.
    """

    _lib.need_cuda(logits, tokens, seq_start, uniforms, draft_logits, scratch)
    x = _rows(logits, "logits")
    r, v = x.shape
    near = None if draft_logits is None else _rows(draft_logits, "draft_logits")
    if near is not None and near.shape != x.shape:
        raise ValueError("verify_drafts: draft_logits must have the shape of logits")
    if tokens.shape != (r,) or tokens.dtype != torch.int32 or not tokens.is_contiguous():
        raise ValueError("verify_drafts: tokens must be contiguous int32, one per row")
    if seq_start.dim() != 1 or seq_start.shape[0] < 2 or seq_start.dtype != torch.int32 or not seq_start.is_contiguous():
        raise ValueError("verify_drafts: seq_start must be contiguous int32 (S+1,)")
    if uniforms.shape != (r, 2) or uniforms.dtype not in (torch.float32, torch.float64) or not uniforms.is_contiguous():
        raise ValueError("verify_drafts: uniforms must be contiguous float32 or float64 (R, 2)")
    near_t = temperature if draft_temperature is None else draft_temperature
    if not 0 < temperature < float("inf") or not 0 < near_t < float("inf"):
        raise ValueError("verify_drafts: temperatures must be positive and finite (greedy: sample_rows and accept_path)")
    if max_window is not None and max_window < 1:
        raise ValueError("verify_drafts: max_window must be positive")
    if any(t is not None and t.device != logits.device for t in (tokens, seq_start, uniforms, near, scratch)):
        raise ValueError("verify_drafts: tensors must be on one device")
    s = seq_start.shape[0] - 1
    lib = _lib.load()
    need = lib.tf_verify_scratch_bytes(r, v)
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
    both = torch.empty((2, s), dtype=torch.int32, device=x.device)
    with _lib.on(x.device):
        _lib.check(lib.tf_verify_rows(x, x.stride(0), near, near.stride(0) if near is not None else 0, tokens, seq_start, uniforms,
                                      int(uniforms.dtype == torch.float64), both[0], both[1], scratch, scratch.numel() * scratch.element_size(),
                                      r, v, s, float(temperature), float(near_t), _lib.stream()), "verify_drafts")
    return both[0], both[1]


__all__ = ["MAX_VOCAB", "verify_drafts"]
