"""The linear layer's plans, without a GPU (where none is, they are those of 256 CUs)."""
import ctypes as C

import pytest
from linear_sizes import SIZES, drawn, plan, variants

from forward_amd import lib


def test_the_tested_sizes_reach_every_variant_that_sizes_choose():
    tested = set().union(*(variants(*s) for s in SIZES))
    missing = {}
    for s in drawn(60000, 3):
        for v in variants(*s) - tested:
            missing.setdefault(v, s)
    assert not missing, missing
    # all of the launchers' tiles, unsplit and split, of each product
    for what in range(3):
        for dtype, tiles in ((lib.F32, {3, 4, 5, 6, 9, 10}), (lib.F16, {0, 1, 2, 3, 4, 5, 6, 9})):
            for split in (False, True):
                assert tiles <= {v[2] for v in tested if v[0] == what and v[1] == dtype and v[5] == split}


def test_both_products_share_a_launch_only_where_one_can_hold_them():
    assert plan(33, 33, 1 << 20, 3, 0, lib.F32, 1).tile_rows > 0
    for m, n, k in ((33, 33, 1 << 28), (33, 33, 1 << 29), (64, 64, (1 << 28) + 8)):      # 2^23 tiles and more of 512 work-items
        assert plan(m, n, k, 3, 0, lib.F32, 1).tile_rows == 0, (m, n, k)


def test_plans_agree_with_the_workspace():
    for m, n, k, on, act in drawn(3000, 5):
        for dtype in (lib.F32, lib.BF16):
            p = plan(m, n, k, 0, 0, dtype, on)
            size = lib.dll.fwdmi_linear_workspace(m, n, k, dtype)
            assert p.splits == 1 or size >= p.splits * m * n * 4
            back = lib.dll.fwdmi_linear_backward_workspace(m, n, k, act, dtype)
            x, w = plan(m, n, k, 1, act, dtype, on), plan(m, n, k, 2, act, dtype, on)
            assert x.splits == 1 or back >= x.splits * m * k * 4
            assert w.splits == 1 or back >= w.splits * n * k * 4


def test_what_is_refused():
    p = lib.LinearPlan()
    ask = lambda *a: lib.dll.fwdmi_linear_plan(*a, C.byref(p))
    assert ask(4, 8, 16, 0, 0, lib.I8, 1) == lib.ERR_UNSUPPORTED
    for bad in ((0, 8, 16, 0, 0), (4, -1, 16, 0, 0), (4, 8, 1 << 31, 0, 0), (4, 8, 16, 4, 0), (4, 8, 16, -1, 0), (4, 8, 16, 0, 9)):
        assert ask(*bad, lib.F16, 1) == lib.ERR_BAD_ARG, bad
    assert lib.dll.fwdmi_linear_plan(4, 8, 16, 0, 0, lib.F16, 1, None) == lib.ERR_BAD_ARG


@pytest.mark.parametrize("k, end", [(96, 0), (98, 1), (97, 1)])
def test_how_the_end_of_the_sum_is_loaded(k, end):
    p = plan(500, 700, k, 0, 0, lib.F32, 1)
    assert p.direct and p.end == (end if k % 4 else 0)
    assert not plan(500, 700, 97, 0, 0, lib.F16, 1).direct                     # lines of an odd number of 16-bit elements
    assert plan(500, 700, 96, 0, 0, lib.F16, 0).direct == 0 and plan(500, 700, 96, 0, 0, lib.F32, 0).direct == 1
