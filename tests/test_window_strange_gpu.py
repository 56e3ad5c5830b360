"""Windowed lane attention where values are not finite: what a row's log-sum-exp and the rows beside it are then."""

import math

import pytest
import torch

from tests.helpers import assert_same_bits
from tests.test_window_gpu import attend, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("h,hk,d", [(24, 4, 256), (16, 2, 128)])
@pytest.mark.parametrize("context", [256, 1000])
@pytest.mark.parametrize("alone", [False, True])
def test_values_that_are_not_finite_leave_the_log_sum_exps(lib, bad, h, hk, d, context, alone):
    """A log-sum-exp depends on keys alone, whether the value lies on a page that all rows see or on one that some see; the rows that see
    it are not finite there, the others keep their bits. One slot and many, few rows (a cluster) and many."""

    lens, widths = ([200], [4]) if alone else ([200, 33, 77, 150], [20, 40, 1, 9])
    window, sinks = 120, 4
    clean = make(21, lens, widths, h, hk, d)
    want, wl = attend(clean, lens, widths, window, sinks, context=context)
    # (slot of sequence 0, the rows of its window that see it): a committed key that all rows see, one that the first ones see, a sink, a window row
    w = widths[0]
    for slot, sees in ((180, range(w)), (200 + 2 - window + 1, range(0, 3)), (2, range(w)), (202, range(2, w))):
        c = make(21, lens, widths, h, hk, d)
        if slot < 200:
            c["v"][int(c["table"][0, slot // 16]), 0, slot % 16, 5] = bad
        else:
            c["v_new"][slot - 200, 0, 5] = bad
        got, lse = attend(c, lens, widths, window, sinks, context=context)
        assert_same_bits(lse, wl, f"slot {slot}")
        spoilt = torch.zeros(got.shape[:2], dtype=torch.bool)
        spoilt[list(sees), :h // hk] = True
        assert not bool(got[..., 5].isfinite()[spoilt.cuda()].any()), slot
        assert_same_bits(got[~spoilt.cuda()], want[~spoilt.cuda()], f"slot {slot}")
