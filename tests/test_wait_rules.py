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


def _prefix_order(pieces):
    """What the products' warp of chunk_tc_kernel<PREFIX> does, in order: ("use", operand)
    issues the product that frees an operand's slot, ("clean", i) waits for masked tile i
    (a piece's last tile).  Operands: K and V of each tile, one after the other."""
    out, first, masked = [], 0, 0
    for nt in pieces:
        scores = lambda j: out.append(("use", first + 2 * j))  # noqa: E731
        scores(0)
        if nt > 1:
            scores(1)
        for j in range(nt):
            if j == nt - 1:
                out.append(("clean", masked))
                masked += 1
            out.append(("use", first + 2 * j + 1))
            if j + 2 < nt:
                scores(j + 2)
        first += 2 * nt
    return out


def test_masked_tiles_of_prefixes_have_barriers_enough():
    """The warps that clean masked tiles may run ahead as far as the ring goes.  A barrier
    that completes a second time before its first completion was waited for looks as if it
    had not: tile i + cleans may only be in the ring once tile i has been waited for."""
    import random
    slots = int(re.search(r"kPrefixSlots = (\d+);", _code("hyq_paged_tc.cuh")).group(1))
    cleans = int(re.search(r"cleans = PREFIX \? (\d+) : 2;", _code("hyq_paged_tc.cu")).group(1))
    rng = random.Random(1)
    for case in ([1] * 12, [2] * 12, [3, 1, 1, 1, 1, 2, 1, 1, 1], *([rng.randint(1, 4) for _ in range(20)] for _ in range(50))):
        order = _prefix_order(case)
        when = {step: n for n, step in enumerate(order)}
        last_v = [2 * sum(case[:i + 1]) - 1 for i in range(len(case))]       # operand of each masked tile
        for i in range(len(case) - cleans):
            freed = last_v[i + cleans] - slots       # whose slot it takes
            assert freed < 0 or when["use", freed] > when["clean", i], (case, i)
