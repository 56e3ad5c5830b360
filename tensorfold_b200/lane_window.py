"""Lane attention with a sliding window and sinks over the paged KV cache.

Beside ``lane_attention.lane_attention``: the same ragged windows of many sequences and the same pages, but a row sees only the
``window`` latest keys and the first ``sinks`` ones, the call costs what those keys cost however long the
sequence is, and it can leave each row's log-sum-exp (what ``lane_evict.attention_mass`` reads). Without a window all keys
are seen. The reference has no counterpart. Chain windows only.
"""

from __future__ import annotations

import torch

from . import _lib
from .lane_attention import PAGE

TILE = 64


def chunk_keys_for(n_seqs: int, heads: int, kv_heads: int, max_window: int, max_context: int, window: int | None = None, sinks: int = 0) -> int:
    """Keys a chunk that ``window_attention`` takes unless it is told: the key axis is cut there, by absolute position, into
    pieces that are attended by themselves and joined."""

    return 512


def window_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                     page_table: torch.Tensor, seq_lens: torch.Tensor, seq_start: torch.Tensor, *, scale: float, max_window: int,
                     max_context: int, window: int | None = None, sinks: int = 0, chunk_keys: int | None = None,
                     scratch: torch.Tensor | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                     gate: torch.Tensor | None = None, packed_out=None) -> torch.Tensor:
    """Attend (R, H, D) queries to each row's sequence: row t of sequence s stands at slot p = seq_lens[s] + t and sees key
    j <= p where p - j < ``window`` or j < ``sinks`` (``window`` None: every j <= p).

    k_new, v_new (R, HK, D) window rows; k_pages, v_pages (pages, HK, 16, D); page_table (S, max_pages), seq_lens (S,),
    seq_start (S+1,) int32 on the device. Table entries of pages that no row sees are never followed, so such pages may have been
    given back (``PagedKV.release_before``). ``max_window`` bounds a sequence's rows, ``max_context`` its keys with the window's
    own; a sequence beyond them is reported through the status word. Rows behind the last sequence (R may exceed
    seq_start[S]) are left as they were in ``out`` and ``lse``.
    ``lse``: float32 (R, H), receives ln(sum exp(score)) of each row and head. ``gate``, ``packed_out``, ``scratch``: as for
    ``lane_attention``. ``chunk_keys``: a multiple of 64; a row's bits depend on it and on the row's own keys, not on the rows
    beside it, so an engine that compares windows with serial steps gives all its calls the same one.
    """

    _lib.need_cuda(q, k_new, v_new, k_pages, v_pages, page_table, seq_lens, seq_start, lse, gate, out, scratch)
    if q.dim() != 3 or k_new.dim() != 3 or k_pages.dim() != 4 or page_table.dim() != 2:
        raise ValueError("unsupported attention shape")
    r, h, d = q.shape
    hk = k_new.shape[1]
    s = seq_lens.shape[0]
    if (r < 1 or k_new.shape != (r, hk, d) or v_new.shape != k_new.shape or d not in (128, 256) or hk < 1 or h % hk or h // hk > 16
            or k_pages.shape[1:] != (hk, PAGE, d) or v_pages.shape != k_pages.shape or page_table.shape[0] != s
            or seq_start.shape != (s + 1,) or seq_lens.dim() != 1):
        raise ValueError("unsupported attention shape")
    for t in (q, k_new, v_new, k_pages, v_pages):
        if t.dtype != torch.bfloat16 or not t.is_contiguous():
            raise ValueError("attention tensors must be contiguous bf16")
    for t in (page_table, seq_lens, seq_start):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError("page_table, seq_lens and seq_start must be contiguous int32")
    if not 0 < scale < float("inf"):
        raise ValueError("scale must be positive and finite")
    if window is not None and window < 1 or sinks < 0 or max_window < 1 or max_context < max_window:
        raise ValueError("window >= 1 (or None), sinks >= 0 and max_context >= max_window >= 1 required")
    if chunk_keys is None:
        chunk_keys = chunk_keys_for(s, h, hk, max_window, max_context, window, sinks)
    if chunk_keys < TILE or chunk_keys % TILE:
        raise ValueError(f"chunk_keys must be a positive multiple of {TILE}")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (r, h) or not lse.is_contiguous()):
        raise ValueError("lse must be contiguous float32 (R, H)")
    if out is not None and (out.dtype != torch.bfloat16 or out.shape != q.shape or not out.is_contiguous()):
        raise ValueError("out must be contiguous bf16 (R, H, D)")
    if gate is not None and (gate.dtype != torch.bfloat16 or gate.shape != (r, h * 2 * d) or gate.stride(1) != 1):
        raise ValueError("gate must be the (R, H * 2 * D) bf16 rows of the q projection")
    if packed_out is not None and (packed_out.m != r or packed_out.k != h * d):
        raise ValueError("packed_out must hold R rows of H * D inputs")
    for t in (k_new, v_new, k_pages, v_pages, page_table, seq_lens, seq_start, lse, out, gate, scratch):
        if t is not None and t.device != q.device:
            raise ValueError("attention tensors must be on one device")
    lib = _lib.load()
    win = 0 if window is None else min(int(window), 1 << 30)
    first = min(int(sinks), 1 << 30) if win else 0
    need = lib.tf_window_scratch_bytes(r, h, d, lib.tf_window_slots(win, first, max_window, max_context, chunk_keys))
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
    if out is None and packed_out is None:
        out = torch.empty_like(q)
    with _lib.on(q.device):
        _lib.check(lib.tf_window_attention(
            q, k_new, v_new, k_pages, v_pages, k_pages.shape[0], page_table, page_table.shape[1], seq_lens, seq_start, out, lse,
            gate, gate.stride(0) if gate is not None else 0, packed_out.data if packed_out is not None else None,
            packed_out.group if packed_out is not None else 64, scratch, scratch.numel() * scratch.element_size(), r, s, max_window,
            max_context, win, first, chunk_keys, h, hk, d, float(scale), _lib.status(q.device).word, _lib.stream()), "window_attention")
    return out if out is not None else packed_out


__all__ = ["chunk_keys_for", "window_attention"]
