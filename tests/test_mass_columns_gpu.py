"""Attention weight per cached key where a block has many tiles: rings that wrap, queries kept over several tiles, runs that begin in the middle of a column
(a layer, KV head and sequence) and go on into the next ones."""

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")


def check(layers, h, hk, d, lens, widths, keep, seed):
    from tensorfold_b200 import _lib, lane_evict

    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
    g, r = h // hk, sum(widths) + 2
    need = [-(-(n + w) // 16) for n, w in zip(lens, widths)]
    count = sum(need) + 3
    order = torch.randperm(count, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need)), -5, dtype=torch.int32, device="cuda")
    at, starts = 0, [0]
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
        starts.append(starts[-1] + widths[s])
    k = rand(layers, count, hk, 16, d).to(BF)
    q = (2 * rand(layers, r, h, d)).to(BF)
    lse = 6 + 2 * torch.rand((layers, r, h), generator=gen, device="cuda")
    mass = torch.rand((layers, count, hk, 16), generator=gen, device="cuda")
    pos = torch.randint(0, 1 << 20, mass.shape, generator=gen, device="cuda", dtype=torch.int32)
    row_pos = torch.randint(0, 1 << 20, (r,), generator=gen, device="cuda", dtype=torch.int32)
    want, want_p = mass.double(), pos.clone()
    tiles = 0
    for s, (n, m) in enumerate(zip(lens, keep)):
        if not m:
            continue
        tiles += -(-(n + m) // 128)
        j = torch.arange(n + m, device="cuda")
        pg, pl = table[s].long()[j // 16], j % 16
        unseen = j > torch.arange(n, n + m, device="cuda").unsqueeze(1)
        for layer in range(layers):
            rows = slice(starts[s], starts[s] + m)
            sc = torch.einsum("tkgd,jkd->kgtj", q[layer, rows].double().reshape(m, hk, g, d), k[layer, pg, :, pl].double()) * d ** -0.5
            e = (sc - lse[layer, rows].double().reshape(m, hk, g).permute(1, 2, 0).unsqueeze(-1)).exp().masked_fill(unseen, 0.0).sum((1, 2))
            old = want[layer, pg, :, pl]
            old[n:] = 0.0
            want[layer, pg, :, pl] = old + e.T
            want_p[layer, pg[n:], :, pl[n:]] = row_pos[rows].reshape(m, 1).expand(m, hk)
    lane_evict.attention_mass(q, lse, k, table, i32(lens), i32(starts), i32(keep), row_pos, mass, pos, scale=d ** -0.5, max_window=max(widths),
                              max_context=max(n + w for n, w in zip(lens, widths)))
    _lib.status(mass.device).raise_if_set()
    # a score off by less than 2^-14 (fp32 sums of 256 products) puts its weight off by that much of itself; the sum of up to 128 x 16 positive
    # terms in fp32 by less than 2^-13 of itself; what is not written stays as it is
    err = (mass.double() - want).abs()
    assert bool((err <= 2.0 ** -12 * want).all()), float((err / want).max())
    assert torch.equal(pos, want_p)
    return layers * hk * tiles


@pytest.mark.parametrize("h,hk,d", [(24, 4, 256), (32, 4, 128), (8, 2, 256), (5, 5, 128)])
@pytest.mark.parametrize("layers", [1, 4])
def test_many_tiles_a_block(lib, h, hk, d, layers):
    lens, widths = [3000, 0, 300, 1777, 128, 2900, 64, 2048, 511, 0, 2600, 127], [8, 4, 3, 1, 8, 2, 6, 5, 8, 2, 7, 1]
    keep = [8, 0, 2, 1, 8, 0, 1, 5, 3, 2, 7, 1]
    assert check(layers, h, hk, d, lens, widths, keep, h + layers) == 89 * layers * hk          # on 148 blocks: up to 12 each


@pytest.mark.parametrize("h,hk,d", [(24, 4, 256), (16, 1, 128)])
def test_many_tiles_and_more_than_128_query_rows(lib, h, hk, d):
    """Query rows in parts of 128, staged anew for every tile, beside sequences whose rows are staged once a column."""

    lens, widths, keep = [2500, 1900, 40, 3000, 700], [40, 3, 60, 30, 100], [37, 3, 60, 22, 100]
    assert check(3, h, hk, d, lens, widths, keep, h) > 148


def test_one_long_column(lib):
    """All blocks in one column, many tiles each."""

    assert check(1, 16, 1, 128, [60000], [5], [5], 3) > 3 * 148


@pytest.mark.parametrize("seqs", [40, 70])
def test_more_sequences_than_a_warp_has_lanes(lib, seqs):
    """The block's share is found over the sequences' tiles, 32 sequences at a time."""

    lens = [(97 * s * s + 31 * s) % 1400 for s in range(seqs)]
    widths = [1 + s % 3 for s in range(seqs)]
    keep = [0 if s % 5 == 1 or 32 <= s < 36 else 1 + s % widths[s] for s in range(seqs)]
    check(2, 12, 2, 128, lens, widths, keep, seqs)
