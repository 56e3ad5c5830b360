"""Host side of the bounded cache and of draft verification: pages given back, chunk sizes, and what the entry points refuse before a launch."""

import ctypes

import pytest
import torch


def kv(pages=20, seqs=2, most=12):
    from tensorfold_b200 import lane_attention as LA

    return LA.PagedKV(1, seqs, pages, 1, 128, most, "cpu")


def held(cache):
    return [int(cache.table_host[s, i]) for s in range(cache.n_seqs) for i in range(cache.owned[s]) if (s, i) not in cache.holes]


def test_pages_out_of_a_window_are_given_back_once():
    cache = kv()
    cache.reserve(0, 150)                                    # 10 pages
    cache.reserve(1, 40)
    assert cache.release_before(0, 100, window=50, sinks=20) == 1       # positions below 51 are out of sight: pages 0..2, of which 0 and 1 hold sinks
    assert cache.release_before(0, 100, window=50, sinks=20) == 0
    assert cache.release_before(0, 140, window=50, sinks=20) == 2
    assert cache.release_before(1, 40, window=50) == 0
    cache.reserve(0, 180)
    assert sorted(held(cache) + cache.free) == list(range(20))          # every page in one place
    cache.release(0)
    cache.release(1)
    assert sorted(cache.free) == list(range(20)) and not cache.holes
    cache.reserve(0, 64)
    assert cache.release_before(0, 63, window=16) == 3


def test_shrunk_pages_are_given_back():
    cache = kv()
    cache.reserve(0, 150)
    assert cache.shrink(0, 64) == 6 and cache.owned[0] == 4
    assert cache.shrink(0, 64) == 0 and cache.shrink(0, 63) == 0 and cache.shrink(0, 48) == 1
    cache.reserve(0, 100)
    assert sorted(held(cache) + cache.free) == list(range(20))
    cache.release_before(0, 100, window=20)
    cache.shrink(0, 17)
    assert sorted(held(cache) + cache.free) == list(range(20))


@pytest.mark.parametrize("seqs", [1, 3, 16, 200])
@pytest.mark.parametrize("heads,kv_heads", [(24, 4), (16, 1), (8, 8)])
@pytest.mark.parametrize("rows", [1, 8, 128, 3000])
@pytest.mark.parametrize("context,window,sinks", [(3000, None, 0), (200000, None, 0), (200000, 1000, 4), (3001, 1, 0)])
def test_chunk_sizes(lib, seqs, heads, kv_heads, rows, context, window, sinks):
    from tensorfold_b200 import lane_window as W

    chunk = W.chunk_keys_for(seqs, heads, kv_heads, rows, context, window, sinks)
    assert chunk >= 128 and chunk % 64 == 0
    slots = lib.tf_window_slots(window or 0, sinks, rows, context, chunk)
    seen = context if window is None else min(context, window + rows - 1)
    assert -(-seen // chunk) <= slots <= -(-context // chunk)
    assert W.scratch_bytes(rows, heads, 128, max_window=rows, max_context=context, window=window, sinks=sinks, chunk_keys=chunk) >= slots * rows * heads * 130 * 4


def test_slots_cover_any_window(lib):
    """Chunks that the rows of a sequence see never share a slot: counted out for small numbers."""

    for window in (1, 63, 64, 65, 200):
        for sinks in (0, 1, 64, 130):
            for rows in (1, 2, 40):
                for chunk in (64, 128):
                    context = 700
                    slots = lib.tf_window_slots(window, sinks, rows, context, chunk)
                    head = min(-(-sinks // chunk), -(-context // chunk))
                    for n in range(0, context - rows + 1, 7):
                        first = max(0, n + 1 - window)
                        chunks = {j // chunk for j in range(first, n + rows)} | {j // chunk for j in range(min(sinks, n + rows))}
                        where = {c if c < head else head + (c - head) % max(slots - head, 1) for c in chunks}
                        assert len(where) == len(chunks) and max(where) < slots, (window, sinks, rows, chunk, n)


def test_launch_counts(lib):
    assert lib.tf_window_launches(1, 1, 1, 32, 24, 4, 256, 1) == 2                 # 128 items: a block each
    assert lib.tf_window_launches(1, 1, 1, 38, 24, 4, 256, 1) == 3                 # 152: some blocks take two
    assert lib.tf_window_launches(128, 16, 8, 128, 24, 4, 256, 1) == 3             # 8192
    assert lib.tf_window_launches(128, 16, 8, 129, 24, 4, 256, 1) == 2
    assert lib.tf_window_launches(128, 16, 100, 20, 24, 4, 256, 1) == 3            # 5 groups of 21 rows
    assert [lib.tf_window_launches(rows, 1, rows, slots, 24, 4, 256, 0) for rows, slots in ((1, 2), (4, 16), (5, 16), (1, 17))] == [1, 1, 2, 2]     # clusters
    assert [lib.tf_window_launches(1, seqs, 1, 1, 24, 4, 256, plain) for seqs, plain in ((2, 1), (2, 0), (60, 1), (60, 0))] == [1, 2, 2, 3]
    assert lib.tf_window_launches(0, 1, 1, 1, 1, 1, 128, 1) == lib.tf_window_launches(1, 1, 1, 1, 34, 2, 128, 1) == lib.tf_window_launches(1, 1 << 15, 1, 1 << 15, 4, 4, 128, 1) == 0
    assert lib.tf_window_launches(1, 1, 1, 74, 24, 4, 128, 1) == 2 and lib.tf_window_launches(1, 1, 1, 75, 24, 4, 128, 1) == 3      # two blocks an SM


def test_refusals_before_any_launch(lib):
    from tensorfold_b200 import _lib

    buf = (ctypes.c_char * 8192)()
    p = (ctypes.addressof(buf) + 255) & ~255
    big = 1 << 40

    def window(q=p, scratch=p, size=big, rows=2, seqs=1, wide=2, context=100, win=10, sinks=0, chunk=64, heads=24, kv_heads=4, d=256, scale=0.1, out=p,
               gate=None, stride=0, group=64, pages=4):
        return lib.tf_window_attention(q, p, p, p, p, pages, p, 8, p, p, out, None, gate, stride, None, group, scratch, size, rows, seqs, wide, context, win,
                                       sinks, chunk, heads, kv_heads, d, scale, None, None)

    for bad in (dict(rows=0), dict(seqs=0), dict(wide=0), dict(context=1), dict(win=-1), dict(sinks=-1), dict(chunk=32), dict(chunk=100), dict(heads=23), dict(heads=68),
                dict(d=64), dict(scale=0.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(out=None), dict(q=None), dict(group=16), dict(gate=p, stride=8),
                dict(pages=0), dict(rows=70000), dict(pages=1 << 30),
                dict(rows=65000, heads=64000, kv_heads=4000), dict(chunk=(1 << 30) + 64)):
        assert window(**bad) == _lib.TF_EINVAL, bad
    assert window(q=p + 2) == window(out=p + 8) == _lib.TF_EALIGN
    assert window(scratch=None) == window(size=64) == _lib.TF_ESCRATCH

    def mass(q=p, layers=1, rows=2, seqs=1, wide=2, context=10, heads=4, kv_heads=2, d=128, scale=1.0):
        return lib.tf_attention_mass(q, p, p, 4, p, 8, p, p, p, p, p, p, layers, rows, seqs, wide, context, heads, kv_heads, d, scale, None, None)

    for bad in (dict(layers=0), dict(rows=0), dict(seqs=0), dict(wide=0), dict(context=1), dict(heads=3), dict(heads=34), dict(d=96), dict(scale=-1.0), dict(q=None),
                dict(layers=300, seqs=300)):
        assert mass(**bad) == _lib.TF_EINVAL, bad
    assert mass(q=p + 4) == _lib.TF_EALIGN

    def evict(k=p, scratch=p, size=big, budget=8, recent=2, sinks=1, context=20, d=128, heads=2, layers=1, mass_at=p):
        return lib.tf_kv_evict(k, p, 4, p, 8, p, p, mass_at, p, p, scratch, size, layers, 1, budget, recent, sinks, context, heads, d, None, None)

    for bad in (dict(budget=0), dict(recent=-1), dict(sinks=-1), dict(recent=8), dict(context=0), dict(d=64), dict(heads=0), dict(layers=0), dict(k=None)):
        assert evict(**bad) == _lib.TF_EINVAL, bad
    assert evict(k=p + 8) == evict(mass_at=p + 4) == _lib.TF_EALIGN
    assert evict(scratch=None) == evict(size=4) == _lib.TF_ESCRATCH

    def verify(x=p, stride=100, near=None, near_stride=0, u=p, f64=0, scratch=p, size=big, rows=2, vocab=100, seqs=1, temp=1.0, near_temp=1.0):
        return lib.tf_verify_rows(x, stride, near, near_stride, p, p, u, f64, p, p, scratch, size, rows, vocab, seqs, temp, near_temp, None)

    for bad in (dict(x=None), dict(stride=99), dict(near=p, near_stride=99), dict(rows=0), dict(rows=40000), dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(seqs=0),
                dict(temp=0.0), dict(temp=float("nan")), dict(near_temp=-1.0), dict(temp=1e9)):
        assert verify(**bad) == _lib.TF_EINVAL, bad
    assert verify(x=p + 1) == verify(u=p + 4, f64=1) == _lib.TF_EALIGN
    assert verify(scratch=None) == verify(size=8) == _lib.TF_ESCRATCH


def test_python_refuses_cpu_tensors(lib):
    from tensorfold_b200 import lane_evict, lane_window, speculative

    x = torch.zeros((2, 4, 128), dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    pages = torch.zeros((1, 3, 4, 16, 128), dtype=torch.bfloat16)
    plane = torch.zeros((1, 3, 4, 16))
    with pytest.raises(ValueError):
        lane_window.window_attention(x, x, x, pages[0], pages[0], i.reshape(1, 2), i[:1], i, scale=1.0, max_window=1, max_context=2)
    with pytest.raises(ValueError):
        lane_evict.attention_mass(x[None], plane[0, 0], pages, i.reshape(1, 2), i[:1], i, i[:1], i, plane, plane.int(), scale=1.0, max_window=1, max_context=2)
    with pytest.raises(ValueError):
        lane_evict.evict(pages, pages, i.reshape(1, 2), i[:1], i[:1], plane, plane.int(), 4, recent=0, max_context=8)
    with pytest.raises(ValueError):
        speculative.verify_drafts(x[0], i, i, torch.zeros((4, 2)))
