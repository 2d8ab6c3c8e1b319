"""The ring of codes in the projection of many rows, followed as the one of the grouped prefill GEMMs is: two sets of convert warps take turns at the stretches, and
an adapter's stretch takes none of the ring, so an odd number of adapters hands every stage from one set to the other at a tile's end. Every wait for a
stage has to know by then that the use before has landed (no GPU needed)."""

import os
import re

import pytest

from tests.test_prefill_raw_ring import walk

with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "drama_rs_b200", "csrc", "proj_rows.cuh")) as _f:
    SRC = _f.read()
NRAW, NA = (int(n) for n in re.search(r"NRAW = (\d+), NA = (\d+);", SRC).groups())
SETS = 2


def test_the_sets_and_the_order_of_the_waits():
    assert "CONV = 8, SET = 4, SETS = CONV / SET" in SRC
    convert = SRC[SRC.index("for (int c = warp >> 2, t = c / seq, g = c % seq; c < total; c += SETS)") : SRC.index("} else if (warp < MMA_WARP) {")]
    # codes: the stage first, then the multiplications that read the operand's columns; an adapter waits for those as well
    assert convert.index("ctl.rawfull[r]") < convert.index("ctl.done[s]") and convert.count("if (use > 0) mbar_wait_ring<DRB_ERR_TMEM>(smem_u32(&ctl.done[s])") == 2


@pytest.mark.parametrize("groups", [1, 2, 3, 5, 6, 16, 17, 63, 64])
@pytest.mark.parametrize("adapters", [0, 1, 2, 3, 4, 7, 80])
def test_every_wait_for_a_stage_is_unambiguous(groups, adapters):
    raws = ([1] * groups + [0] * adapters) * 6
    assert walk(raws, NRAW, NA, SETS, [False] * len(raws)) == []


def test_a_shorter_ring_would_not_be():
    raws = ([1] * 16 + [0]) * 6
    assert walk(raws, 3, NA, SETS, [False] * len(raws))
