"""``window_attention`` over the whole cache and ``lane_attention``, whose place it takes in a state with a budget: the same attention."""

import pytest
import torch

from tests.test_window_gpu import attend, make, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("h,hk,d", [(24, 4, 256), (16, 2, 128), (6, 1, 256)])
@pytest.mark.parametrize("lens,widths", [([700], [1]), ([0, 300, 1500, 15], [3, 8, 1, 20]), ([130], [128])])
def test_both_are_near_the_same(lib, h, hk, d, lens, widths):
    from tensorfold_b200 import lane_attention as LA

    c = make(h + len(lens), lens, widths, h, hk, d)
    got, _ = attend(c, lens, widths, None, 0)
    g = {n: t.cuda() for n, t in c.items()}
    nkeys = torch.tensor([n + t + 1 for n, w in zip(lens, widths) for t in range(w)], dtype=torch.int32, device="cuda")
    want = LA.lane_attention(g["q"], g["k_new"], g["v_new"], g["k"], g["v"], g["table"], g["lens"], g["start"], nkeys, scale=d ** -0.5, max_window=max(widths),
                             max_chunks=LA.chunks_for(int(nkeys.max())))
    for s, w in enumerate(widths):
        r0 = int(c["start"][s])
        exact, _, size = plain(c, s, lens, widths, None, 0)
        # each of the two: weights rounded to bf16 (2^-8 of each term), scores off by less than 2^-14, the result rounded once
        bound = 2 * ((2.0 ** -8 + 2.0 ** -12) * size + 2.0 ** -8 * exact.abs())
        assert bool(((got[r0:r0 + w].double() - want[r0:r0 + w].double()).abs().cpu() <= bound).all())
