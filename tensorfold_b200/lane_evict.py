"""A bounded KV cache: the attention weight every cached key has received, and eviction by it.

Beside ``lane_attention.kv_commit``: after a commit ``attention_mass`` adds the weight that the kept rows gave each cached key
of each layer and KV head (the attention's log-sum-exps, ``lane_window.window_attention(lse=...)``, make a
second softmax unnecessary), and ``evict`` cuts sequences that outgrew their budget back to it: the first tokens and the latest ones
stay, and of the others those that received the most. A layer's KV heads choose by themselves; all keep the same number of
slots, so the page table stays common. Keys carry their rotation: the slots' order does not matter, and eviction moves as few
rows as it can. The reference has no counterpart.
"""

from __future__ import annotations

import torch

from . import _lib


def attention_mass(q: torch.Tensor, lse: torch.Tensor, k_pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                   seq_start: torch.Tensor, keep: torch.Tensor, row_pos: torch.Tensor, mass: torch.Tensor, pos: torch.Tensor, *, scale: float,
                   max_window: int, max_context: int) -> None:
    """Bring ``mass`` and ``pos`` up to date after ``kv_commit`` kept the first keep[s] rows of every window, all layers at once.

    q (layers, R, H, D) bf16 and lse (layers, R, H) float32: the queries and log-sum-exps of the attention over the whole cache;
    k_pages (layers, pages, HK, 16, D); seq_lens (S,): the lengths before the commit; row_pos (R,): each row's position in the text;
    mass float32 and pos int32 (layers, pages, HK, 16), a cell per cached key. Every key gains the sum, over the kept rows that
    see it and its KV head's query heads, of exp(scale q . k - lse); the keys that the commit brought start at that sum and
    take their row's position. ``max_window`` bounds a sequence's rows, ``max_context`` its slots after the commit; a sequence beyond
    them is reported through the status word and left as it was.
    """

    _lib.need_cuda(q)
    _lib.host().attention_mass(q, lse, k_pages, page_table, seq_lens, seq_start, keep, row_pos, mass, pos, scale, max_window, max_context,
                               _lib.status(q.device).word)


def scratch_bytes(layers: int, n_seqs: int, kv_heads: int, budget: int, max_context: int) -> int:
    return int(_lib.load().tf_evict_scratch_bytes(layers, n_seqs, kv_heads, budget, max_context))


def evict(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, next_pos: torch.Tensor, mass: torch.Tensor,
          pos: torch.Tensor, budget: int, *, recent: int, sinks: int = 0, max_context: int, scratch: torch.Tensor | None = None) -> torch.Tensor:
    """Cut every sequence of more than ``budget`` slots back to it, in every layer and KV head; returns how many slots each of them
    moved, (layers, S, HK) int32.

    Kept: slots whose position is below ``sinks`` or at least next_pos[s] - ``recent`` (next_pos (S,): the position that the
    sequence's next token takes), then those of the largest mass, ties to the lower slot. The i-th kept slot at or above the budget moves
    into the i-th evicted slot below it, with its mass and position; nothing else is written. The caller then counts
    min(length, budget) slots for the sequence (``PagedKV.shrink`` gives the pages above back). ``seq_lens`` itself is not written.
    Pages must belong to one sequence. ``max_context`` bounds the slots of a sequence; ``scratch``: ``scratch_bytes``.
    """

    _lib.need_cuda(k_pages)
    return _lib.host().evict(k_pages, v_pages, page_table, seq_lens, next_pos, mass, pos, budget, recent, sinks, max_context, scratch,
                             _lib.status(k_pages.device).word)


__all__ = ["attention_mass", "evict", "scratch_bytes"]
