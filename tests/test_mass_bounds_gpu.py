"""What ``attention_mass`` was not called for is reported and left as it was."""

import pytest
import torch

from tests.helpers import assert_same_bits
from tests.test_evict_gpu import cache, cells, i32

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def test_a_sequence_of_more_rows_than_max_window(lib):
    from tensorfold_b200 import _lib, lane_evict

    lens, widths, keep, h, hk, d = [40, 300, 7], [3, 9, 4], [3, 9, 4], 8, 2, 128
    table, k, _, mass, pos, gen = cache(2, 1, [n + w for n, w in zip(lens, widths)], hk, d)
    q, lse = torch.randn((1, 16, h, d), generator=gen).to(BF).cuda(), 5 + torch.rand((1, 16, h), generator=gen).cuda()
    start, row_pos = i32([0, 3, 12, 16]).cuda(), torch.arange(16, dtype=torch.int32).cuda()

    def call(most, kept):
        m, p = mass.cuda(), pos.cuda()
        lane_evict.attention_mass(q, lse, k.cuda(), table.cuda(), i32(lens).cuda(), start, i32(kept).cuda(), row_pos, m, p, scale=0.1, max_window=most,
                                  max_context=309)
        return m, p

    status = _lib.status(q.device)
    status.raise_if_set()
    want = call(9, [3, 0, 4])
    status.raise_if_set()
    got = call(8, keep)
    with pytest.raises(RuntimeError):
        status.raise_if_set()
    for a, b in zip(got, want):
        assert_same_bits(a, b)
    assert bool((call(9, keep)[0] != want[0]).any())
    status.raise_if_set()
    call(8, [3, 0, 4])                                       # nothing kept of it: nothing to be done, nothing to report
    status.raise_if_set()
