"""Learned type vectors without a GPU: what their calls plan and refuse at the ends of their ranges."""
import ctypes

import pytest


def test_rows_of_a_thread_begin_alike(lib):
    """A thread of a layer norm copies whole pieces of 16 bytes and keeps the place in them at which its first row begins: where rows do not
    begin on 16 bytes, what it jumps by has to be a multiple of the values that 16 bytes hold, or it has one row alone."""
    rows = list(range(1, 20)) + [31, 32, 33, 64, 127, 128, 129, 147, 148, 149, 295, 296, 297, 443, 444, 445, 591, 592, 593, 600, 888, 889, 1184,
                                 1185, 2367, 2368, 2400, 4736, 5000, 9471, 9472, 20000]
    plan = (ctypes.c_uint * 5)()
    broken = []
    for slack in (3, 7):
        for width in range(1, 8193):
            for n in rows:
                lib.lmg_norm_plan(n, width, slack, plan)
                wide, at_once, times, forward, backward = plan
                if wide:
                    continue
                assert times == -(-n // at_once) and 1 <= forward <= times and 1 <= backward <= times
                # the jump in values is at_once * blocks * ld, for any ld
                broken += [(slack, width, n, b) for b in (forward, backward) if b < times and at_once * b % (slack + 1)]
    assert not broken, (len(broken), broken[:5])


@pytest.mark.parametrize("slack", [0, 3, 7])
def test_workspace_covers_every_alignment(lib, slack):
    from libmolgrid_b200 import _cabi
    plan = (ctypes.c_uint * 5)()
    for width in (1, 28, 64, 505, 506, 1001, 4096, 8185, 8192, 9000):
        for n in (1, 2, 3, 4, 5, 100, 1000, 20000):
            lib.lmg_norm_plan(n, width, slack, plan)
            assert lib.lmg_vectors_workspace_bytes(_cabi.OP_LAYER_NORM_BACKWARD, n, 0, width) >= 256 + plan[4] * 2 * width * 4


def test_draws_go_with_type_indices():
    import torch
    import libmolgrid_b200 as lmg
    with pytest.raises(ValueError):
        lmg.Coords2Grid(lmg.GridMaker(0.5, 5.5))(torch.zeros(2, 4, 3), torch.zeros(2, 4, 2), torch.ones(2, 4), draw=(1, 0))
    assert lmg.Dropout(0.0).draw() is None and lmg.TypeVectors(3, 2, p=0.5).eval().draw() is None
