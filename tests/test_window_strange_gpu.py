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


@pytest.mark.parametrize("h,hk,d", [(24, 4, 256), (16, 2, 128)])
@pytest.mark.parametrize("context", [256, 1000])
@pytest.mark.parametrize("alone", [False, True])
@pytest.mark.parametrize("number", [-1, 10 ** 6])
def test_rows_that_see_a_page_that_is_none(lib, h, hk, d, context, alone, number):
    """Reported, and NaN rather than a softmax in which the missing keys score 0; rows that do not see it keep their bits."""

    from tensorfold_b200 import _lib, lane_window

    lens, widths = ([200], [4]) if alone else ([200, 33, 77, 150], [20, 40, 1, 9])
    window, sinks = 120, 4
    clean = make(21, lens, widths, h, hk, d)
    want, wl = attend(clean, lens, widths, window, sinks, context=context)
    # (page of sequence 0, the rows of its window that see it): in the middle, the last of the window (keys 80 to 95), the sinks', the last committed one
    w = widths[0]
    for page, sees in ((9, range(w)), (5, range(min(w, 15))), (0, range(w)), (12, range(w))):
        c = make(21, lens, widths, h, hk, d)
        c["table"][0, page] = number
        out, lse = torch.full_like(want, 55.0), torch.full_like(wl, 77.0)
        g = {n: t.cuda() for n, t in c.items()}
        lane_window.window_attention(g["q"], g["k_new"], g["v_new"], g["k"], g["v"], g["table"], g["lens"], g["start"], scale=d ** -0.5, max_window=max(widths),
                                     max_context=context, window=window, sinks=sinks, chunk_keys=128, lse=lse, out=out)
        with pytest.raises(RuntimeError):
            _lib.status(out.device).raise_if_set()
        lost = torch.zeros(want.shape[0], dtype=torch.bool)
        lost[list(sees)] = True
        lost = lost.cuda()
        assert bool(out[lost].isnan().all()) and bool(lse[lost].isnan().all()), page
        assert_same_bits(out[~lost], want[~lost], f"page {page}")
        assert_same_bits(lse[~lost], wl[~lost], f"page {page}")
