"""Rules of the 8-bit cache's kernels that no run can show: a wait that runs out
does so by each lane's own clock, and making one run out on a GPU would need a
broken kernel; a load through the read-only path sees old bytes once in a long
while or never.  So the source is read."""

import os
import re

import furnace_b200 as fz

KVQ8 = os.path.join(os.path.dirname(fz.__file__), "csrc", "kvq8.cuh")


def _code():
    with open(KVQ8) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def _rows_kernel():
    code = _code()
    body = code[code.index("k_kvq8_rows(const __grid_constant__"):]
    return body[:body.index("\n}\n")]


def _statements(code):
    """Statements that wait on a barrier (the helper's own definition aside)."""
    out = []
    for s in re.split(r"[;{}]", code):
        if re.search(r"\b(mbar_wait|wait)\(", s) and "auto wait" not in s and "reinterpret_cast" not in s:
            out.append(" ".join(s.split()))
    return out


def test_every_wait_of_a_warp_ends_for_all_its_lanes_alike():
    """What follows a wait uses the whole warp (tensor memory loads, shuffles,
    __syncwarp), so lanes of a warp must never come to different ends: the
    result goes through __all_sync.  The one thread that issues the products is
    alone, and each of its waits decides what it does next."""
    body = _rows_kernel()
    lo = body.index("if (warp == 15) {\n    if (lane == 0) {")
    hi = body.index("} else if (warp >= 12) {")
    alone, warps = _statements(body[lo:hi]), _statements(body[:lo] + body[hi:])
    assert len(alone) >= 5 and len(warps) >= 6
    for s in warps:
        assert "__all_sync(0xffffffffu," in s, s
        assert re.match(r"(if \(.*\) )?(bool )?ok = ", s), s
    for s in alone:
        assert re.search(r"\bok = ", s), s


def test_a_wait_that_ran_out_is_reported():
    body = _rows_kernel()
    end = body[body.rindex("__syncthreads()") - 200:]
    assert "if (!ok && lane == 0) atomicOr(a.c.status, KQ_TIMEOUT)" in end


def test_nothing_is_read_through_the_read_only_path():
    """The kernel before may still be writing the cache, the rows and the
    lengths while these kernels are resident."""
    code = _code()
    assert "__ldg" not in code and ".nc" not in code
    assert not re.search(r"const [\w:]+\s*\*\s*__restrict__", code)


def _slots(segments, pages, runs):
    """(run, slot) of every piece that a step with run records writes, as
    k_kvq8_split cuts them: a segment costs its pages and 2."""
    size = pages + 2
    total = segments * size
    per = (total + 2 * runs - 1) // (2 * runs) * 2
    out = []
    for run in range(runs):
        w0, w1 = min(per * run, total), min(per * run + per, total)
        w = w0
        while w < w1:
            u0 = w % size
            u1 = min(size, u0 + w1 - w)
            if max(u1, 2) > max(u0, 2):
                out.append((run, w != w0))
            w += u1 - u0
    return out


def test_a_run_of_a_decode_step_has_room_for_its_pieces():
    """As long as there are no more segments than runs; a step with more is
    refused."""
    assert len(_slots(900, 1, 444)) != len(set(_slots(900, 1, 444)))  # why it has to be
    for segments in (1, 2, 7, 8, 64, 221, 222, 223, 300, 443, 444):
        for pages in (1, 2, 3, 4, 5, 31, 32, 64, 1001):
            runs = min(segments * (pages + 2), 444)
            pieces = _slots(segments, pages, runs)
            assert len(pieces) == len(set(pieces)), (segments, pages)
    code = _code()
    assert "a.runs && a.c.nkv * ((a.c.group + 7) / 8) > kvq8_runs(a.c, a.b)" in code
