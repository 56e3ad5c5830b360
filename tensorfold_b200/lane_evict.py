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
from .lane_attention import PAGE


def _planes(k_pages: torch.Tensor, mass: torch.Tensor, pos: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor) -> tuple:
    if k_pages.dim() != 5 or k_pages.shape[3] != PAGE or k_pages.shape[4] not in (128, 256) or k_pages.dtype != torch.bfloat16 or not k_pages.is_contiguous():
        raise ValueError("the pages must be contiguous bf16 (layers, pages, HK, 16, D), D 128 or 256")
    for t, dtype in ((mass, torch.float32), (pos, torch.int32)):
        if t.shape != k_pages.shape[:4] or t.dtype != dtype or not t.is_contiguous():
            raise ValueError("mass must be contiguous float32 and pos int32, (layers, pages, HK, 16)")
    if page_table.dim() != 2 or seq_lens.dim() != 1 or page_table.shape[0] != seq_lens.shape[0] or seq_lens.shape[0] < 1:
        raise ValueError("page_table must be (S, max_pages) and seq_lens (S,)")
    return k_pages.shape


def _int32(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError("page_table, lengths, positions and counts must be contiguous int32")


def _same_device(first: torch.Tensor, *tensors: torch.Tensor) -> None:
    _lib.need_cuda(first, *tensors)
    if any(t is not None and t.device != first.device for t in tensors):
        raise ValueError("cache tensors must be on one device")


def attention_mass(q: torch.Tensor, lse: torch.Tensor, k_pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                   seq_start: torch.Tensor, keep: torch.Tensor, row_pos: torch.Tensor, mass: torch.Tensor, pos: torch.Tensor, *, scale: float,
                   max_window: int, max_context: int) -> None:
    """Bring ``mass`` and ``pos`` up to date after ``kv_commit`` kept the first keep[s] rows of every window, all layers at once.

    q (layers, R, H, D) bf16 and lse (layers, R, H) float32: the queries and log-sum-exps of the attention over the whole cache;
    k_pages (layers, pages, HK, 16, D); seq_lens (S,): the lengths before the commit; row_pos (R,): each row's position in the text;
    mass float32 and pos int32 (layers, pages, HK, 16), a cell per cached key. Every key gains the sum, over the kept rows that
    see it and its KV head's query heads, of exp(scale q . k - lse); the keys that the commit brought start at that sum and
    take their row's position. ``max_window`` bounds a sequence's rows, ``max_context`` its slots after the commit.
    """

    _same_device(q, lse, k_pages, page_table, seq_lens, seq_start, keep, row_pos, mass, pos)
    layers, pages, hk, _, d = _planes(k_pages, mass, pos, page_table, seq_lens)
    _int32(page_table, seq_lens, seq_start, keep, row_pos)
    s = seq_lens.shape[0]
    if q.dim() != 4 or q.shape[0] != layers or q.shape[1] < 1 or q.shape[3] != d or q.dtype != torch.bfloat16 or not q.is_contiguous():
        raise ValueError("q must be contiguous bf16 (layers, R, H, D)")
    r, h = q.shape[1:3]
    if h < 1 or h % hk or h // hk > 16:
        raise ValueError("H must be a multiple of HK, at most 16 heads a KV head")
    if lse.shape != (layers, r, h) or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError("lse must be contiguous float32 (layers, R, H)")
    if seq_start.shape != (s + 1,) or keep.shape != (s,) or row_pos.shape != (r,):
        raise ValueError("seq_start (S+1,), keep (S,) and row_pos (R,) required")
    if not 0 < scale < float("inf") or max_window < 1 or max_context < max_window:
        raise ValueError("scale must be positive and finite, max_context >= max_window >= 1")
    with _lib.on(q.device):
        _lib.check(_lib.load().tf_attention_mass(q, lse, k_pages, pages, page_table, page_table.shape[1], seq_lens, seq_start, keep, row_pos, mass,
                                                 pos, layers, r, s, max_window, max_context, h, hk, d, float(scale), _lib.status(q.device).word,
                                                 _lib.stream()), "attention_mass")


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

    _same_device(k_pages, v_pages, page_table, seq_lens, next_pos, mass, pos, scratch)
    layers, pages, hk, _, d = _planes(k_pages, mass, pos, page_table, seq_lens)
    _int32(page_table, seq_lens, next_pos)
    s = seq_lens.shape[0]
    if v_pages.shape != k_pages.shape or v_pages.dtype != torch.bfloat16 or not v_pages.is_contiguous() or next_pos.shape != (s,):
        raise ValueError("v_pages must match k_pages and next_pos be (S,)")
    if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget or max_context < 1:
        raise ValueError("budget >= recent + sinks, all non-negative, budget and max_context at least 1")
    lib = _lib.load()
    need = lib.tf_evict_scratch_bytes(layers, s, hk, budget, max_context)
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.uint8, device=k_pages.device)
    moved = torch.empty((layers, s, hk), dtype=torch.int32, device=k_pages.device)
    with _lib.on(k_pages.device):
        _lib.check(lib.tf_kv_evict(k_pages, v_pages, pages, page_table, page_table.shape[1], seq_lens, next_pos, mass, pos, moved, scratch,
                                   scratch.numel() * scratch.element_size(), layers, s, budget, recent, sinks, max_context, hk, d,
                                   _lib.status(k_pages.device).word, _lib.stream()), "evict")
    return moved


__all__ = ["attention_mass", "evict", "scratch_bytes"]
