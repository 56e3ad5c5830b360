"""Lane attention with a sliding window and sinks over the paged KV cache.

Beside ``lane_attention.lane_attention``: the same ragged windows of many sequences and the same pages, but a row sees only the
``window`` latest keys and the first ``sinks`` ones, the call costs what those keys cost however long the
sequence is, and it can leave each row's log-sum-exp (what ``lane_evict.attention_mass`` reads). Without a window all keys
are seen. The reference has no counterpart. Chain windows only.
"""

from __future__ import annotations

import torch

from . import _lib


def chunk_keys_for(n_seqs: int, heads: int, kv_heads: int, max_window: int, max_context: int, window: int | None = None, sinks: int = 0) -> int:
    """Keys a chunk that ``window_attention`` takes unless it is told: the key axis is cut there, by absolute position, into
    pieces that are attended by themselves and joined."""

    chunk = _lib.load().tf_window_chunk_keys(n_seqs, heads, kv_heads, max_window, max_context, 0 if window is None else min(window, 1 << 30), min(sinks, 1 << 30))
    if chunk < 1:
        raise ValueError("at least one sequence, KV head and row, heads >= kv_heads and max_context >= max_window >= 1 required")
    return chunk


def scratch_bytes(rows: int, heads: int, head_dim: int, *, max_window: int, max_context: int, window: int | None, sinks: int, chunk_keys: int) -> int:
    """Bytes of ``window_attention``'s scratch."""

    lib = _lib.load()
    slots = lib.tf_window_slots(0 if window is None else min(window, 1 << 30), sinks if window is not None else 0, max_window, max_context, chunk_keys)
    return int(lib.tf_window_scratch_bytes(rows, heads, head_dim, slots))


def window_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                     page_table: torch.Tensor, seq_lens: torch.Tensor, seq_start: torch.Tensor, *, scale: float, max_window: int,
                     max_context: int, window: int | None = None, sinks: int = 0, chunk_keys: int | None = None,
                     scratch: torch.Tensor | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                     gate: torch.Tensor | None = None, packed_out=None) -> torch.Tensor:
    """Attend (R, H, D) queries to each row's sequence: row t of sequence s stands at slot p = seq_lens[s] + t and sees key
    j <= p where p - j < ``window`` or j < ``sinks`` (``window`` None: every j <= p).

    Softmax weights are rounded to bf16 for their product with V, as in ``lane_attention``; scores, sums and log-sum-exps are float32.

    k_new, v_new (R, HK, D) window rows; k_pages, v_pages (pages, HK, 16, D); page_table (S, max_pages), seq_lens (S,),
    seq_start (S+1,) int32 on the device. Table entries of pages that no row sees are never followed, so such pages may have been
    given back (``PagedKV.release_before``). ``max_window`` bounds a sequence's rows, ``max_context`` its keys with the window's
    own; a sequence beyond them is reported through the status word, and so is a page number that is none on a page that a row sees, which
    makes the row NaN. Rows behind the last sequence (R may exceed
    seq_start[S]) are left as they were in ``out`` and ``lse``.
    ``lse``: float32 (R, H), receives ln(sum exp(score)) of each row and head. ``gate``, ``packed_out``, ``scratch``: as for
    ``lane_attention``. ``chunk_keys``: a multiple of 64; a row's bits depend on it and on the row's own keys, not on the rows
    beside it, so an engine that compares windows with serial steps gives all its calls the same one.
    """

    _lib.need_cuda(q)
    if packed_out is not None and (q.dim() != 3 or packed_out.m != q.shape[0] or packed_out.k != q.shape[1] * q.shape[2]):
        raise ValueError("packed_out must hold R rows of H * D inputs")
    if window is not None and window < 1 or sinks < 0 or chunk_keys is not None and chunk_keys < 1:
        raise ValueError("window >= 1 (or None), sinks >= 0 and chunk_keys >= 1 (or None) required")
    res = _lib.host().window_attention(q, k_new, v_new, k_pages, v_pages, page_table, seq_lens, seq_start, scale, max_window, max_context,
                                       0 if window is None else min(window, 1 << 30), min(sinks, 1 << 30) if window is not None else 0, chunk_keys or 0, scratch, out,
                                       lse, gate,
                                       packed_out.data if packed_out is not None else None, packed_out.group if packed_out is not None else 64,
                                       _lib.status(q.device).word)
    return packed_out if res is None else res


__all__ = ["chunk_keys_for", "scratch_bytes", "window_attention"]
