"""Lane attention with a sliding window and sinks over the paged KV cache.

Beside ``lane_attention.lane_attention``: the same ragged windows of many sequences and the same pages, but a row sees only the
``window`` latest keys and the first ``sinks`` ones, the call costs what those keys cost however long the
sequence is, and it can leave each row's log-sum-exp (what ``lane_evict.attention_mass`` reads). Without a window all keys
are seen. The reference has no counterpart. Chain windows only.
"""

from __future__ import annotations

import math

import torch

from . import _lib


def chunk_keys_for(n_seqs: int, heads: int, kv_heads: int, max_window: int, max_context: int, window: int | None = None, sinks: int = 0) -> int:
    """Keys a chunk that ``window_attention`` takes unless it is told: the key axis is cut there, by absolute position, into
    pieces that are attended by themselves and joined.

    Few columns (sequence, KV head, group of up to 128 query rows): as many chunks as leave the SMs one each, but not below the size at
    which a chunk's tiles (0.95 us for 64 keys) and the join (0.36 us a chunk) cost the same, and one chunk where that saves
    the join for few tiles more (300 rows of up to 400 keys: 16.8 us in one, 21.1 in two). More columns: a quarter of what a group sees, so that the
    chunks can be dealt out evenly (16 x 4 columns of 4100 keys: 59.1 us in chunks of 1024, 59.6 of 2048, 64.8 of 512, 77 of 4096; with heads
    of 128 38.7, 48.7, 43.3 and 71.6). Very many, as for a prompt's rows: one chunk, without partials and join, where a group sees few
    keys (362 columns of 1040 keys: 45.5 us, 57 in chunks of 2048; 576 of 4000: 222 and 284), else 2048 (376 columns of 17500
    keys: 511 us, 643 in one chunk, whose columns do not divide evenly).
    """

    if min(n_seqs, kv_heads, max_window) < 1 or heads < kv_heads or max_context < max_window:
        raise ValueError("at least one sequence, KV head and row, heads >= kv_heads and max_context >= max_window >= 1 required")
    rows = max(1, min(max_window, 128 // (heads // kv_heads)))
    columns = n_seqs * kv_heads * -(-max_window // rows)
    keys = max_context if window is None else min(max_context, window + rows - 1)
    whole = -(-max(max_context, 128) // 64) * 64
    spare = 148 // columns - (0 if window is None else 1 + (sinks > 0))       # a window lies across one chunk more, sinks have their own
    if spare >= 1:
        chunk = -(-max(128, math.isqrt(24 * keys), -(-keys // spare)) // 64) * 64
        return whole if whole - chunk <= 256 else chunk
    if columns < 222:
        return min(max(-(-keys // 256) * 64, 512), 2048)
    return whole if keys <= 4096 else 2048


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

    k_new, v_new (R, HK, D) window rows; k_pages, v_pages (pages, HK, 16, D); page_table (S, max_pages), seq_lens (S,),
    seq_start (S+1,) int32 on the device. Table entries of pages that no row sees are never followed, so such pages may have been
    given back (``PagedKV.release_before``). ``max_window`` bounds a sequence's rows, ``max_context`` its keys with the window's
    own; a sequence beyond them is reported through the status word. Rows behind the last sequence (R may exceed
    seq_start[S]) are left as they were in ``out`` and ``lse``.
    ``lse``: float32 (R, H), receives ln(sum exp(score)) of each row and head. ``gate``, ``packed_out``, ``scratch``: as for
    ``lane_attention``. ``chunk_keys``: a multiple of 64; a row's bits depend on it and on the row's own keys, not on the rows
    beside it, so an engine that compares windows with serial steps gives all its calls the same one.
    """

    _lib.need_cuda(q)
    if q.dim() != 3 or k_new.dim() != 3 or seq_lens.dim() != 1:
        raise ValueError("unsupported attention shape")
    if packed_out is not None and (packed_out.m != q.shape[0] or packed_out.k != q.shape[1] * q.shape[2]):
        raise ValueError("packed_out must hold R rows of H * D inputs")
    if window is not None and window < 1 or sinks < 0:
        raise ValueError("window >= 1 (or None) and sinks >= 0 required")
    if chunk_keys is None:
        chunk_keys = chunk_keys_for(seq_lens.shape[0], q.shape[1], k_new.shape[1], max_window, max_context, window, sinks)
    res = _lib.host().window_attention(q, k_new, v_new, k_pages, v_pages, page_table, seq_lens, seq_start, scale, max_window, max_context,
                                       0 if window is None else min(window, 1 << 30), min(sinks, 1 << 30) if window is not None else 0, chunk_keys, scratch, out, lse, gate,
                                       packed_out.data if packed_out is not None else None, packed_out.group if packed_out is not None else 64,
                                       _lib.status(q.device).word)
    return packed_out if res is None else res


__all__ = ["chunk_keys_for", "scratch_bytes", "window_attention"]
