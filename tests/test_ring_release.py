"""When a stage of a ring goes back to the bulk and tensor copies (no GPU needed).

A load from shared memory has only been queued when the next instruction issues, and an arrival on an mbarrier does not stand in that queue; the
copy that it lets in writes through another proxy. So between the last read of a stage and its arrival there has to be a use of what was read that
keeps its place (the store into tensor memory), or the fence between the proxies. Read from the source: on the GPU a late load showed in
one call of two of one size and never in others."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "drama_rs_b200", "csrc")
ORDERED = ("tmem_st32(", "reads_before_copies();")


def source(name: str) -> str:
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def between(text: str, read: str, release: str) -> list[str]:
    """What stands between each release and the last read before it."""
    found = []
    for m in re.finditer(re.escape(release), text):
        at = text.rfind(read, 0, m.start())
        assert at >= 0, (read, release)
        found.append(text[at : m.start()])
    return found


@pytest.mark.parametrize("file,read,release,places", [("proj_rows.cuh", "(raw + r * RAW_BYTES", "mbar_arrive(&ctl.rawempty[r])", 1),
                                                      ("moe_prefill_tc.cuh", "lds128(xa", "mbar_arrive(&ctl.rawempty[rr.i])", 1),
                                                      ("moe_prefill_tc.cuh", "(xp + piece(", "mbar_arrive(&ctl.rawempty[sa])", 1),
                                                      ("stack_decode.cuh", "dot32_q4_i(gr[lane]", "bar_arrive<THREADS>(BAR_GU)", 2),
                                                      ("stack_decode.cuh", "(dst + TOPK * D_EXPERT + (size_t)warp", "bar_arrive<THREADS>(BAR_DN)", 1)])
def test_a_stage_goes_back_behind_the_use_of_its_reads(file, read, release, places):
    texts = between(source(file), read, release)
    assert len(texts) == places
    for t in texts:
        assert any(o in t for o in ORDERED), t


def test_a_gemvs_stage_goes_back_by_an_arrival_that_waits_for_the_reads():
    """There the address of the arrival is made from what was read: from all pieces of a row, and from the scales unless the slot that they lie in is
    filled again a tile later."""
    text = source("gemv.cuh")
    assert "mbar_arrive(&ctl.empty" not in text and text.count("mbar_arrive_behind(") == 2
    calls = re.findall(r" release\((.*)\);", text)
    assert len(calls) == 2 and all(w in calls[0] for w in ("v0.x", "v1.x", "w0.x", "w1.x", "sc0", "sc1")), calls
    assert all(w in calls[1] for w in ("a0", "a1"))
    assert "+ (NSEG == 2 ? 2 : 0)" in text  # the slots' count, by which two segments do without the scales


def test_the_scan_sees_an_arrival_between_the_reads_and_their_use():
    late = "v = *(raw + r * RAW_BYTES); sync(); mbar_arrive(&ctl.rawempty[r]); tmem_st32(a, v);"
    (text,) = between(late, "(raw + r * RAW_BYTES", "mbar_arrive(&ctl.rawempty[r])")
    assert not any(o in text for o in ORDERED)
