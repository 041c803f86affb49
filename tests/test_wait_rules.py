"""Rules of the kernels whose waits have a limit, read off their sources: what a
warp does that gave up cannot be provoked on a GPU."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hy_mt_rs_b200", "csrc")
SOURCES = sorted(os.path.basename(f) for f in glob.glob(os.path.join(CSRC, "hyq_paged_tc*.cu*")))


def _code(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_there_are_sources():
    assert {"hyq_paged_tc.cu", "hyq_paged_tc32.cu", "hyq_paged_tc8.cu", "hyq_paged_tc.cuh"} <= set(SOURCES)


@pytest.mark.parametrize("name", SOURCES)
def test_no_barrier_waits_for_a_warp_that_gave_up(name):
    """A warp whose wait ran out leaves its loop, and a named barrier has no limit: one
    among such waits has to carry the warps' verdicts (bar_red_and), so that all of
    them leave, and what it says has to be heeded."""
    code = _code(name)
    assert "warp_wait(" in code
    assert not re.search(r"bar\.sync|barrier\.sync|bar_sync_named", code)
    for use in re.finditer(r"[^\n]*bar_red_and\([^\n]*\n[^\n]*\n", code):
        assert re.search(r"ok = bar_red_and\(\d+, \d+, ok\);\s*if \(!ok\) break;", use.group()), use.group()


def test_loaders_of_codes_meet_at_their_barrier():
    """Between two of the loaders' barriers no warp leaves the loop."""
    body = _code("hyq_paged_tc8.cu").split("for (int i = 0; i < tiles; ++i) {", 1)[1].split("cp.async.wait_all", 1)[0]
    assert len(re.findall(r"\bbreak;", body)) == body.count("bar_red_and(") == 1
    assert "return" not in re.sub(r"if \(!ok\) return;\s*ask_values", "", body)    # (ask()'s own)
