"""Calls around the edges of the 8-bit paged KV cache."""

import numpy as np
import pytest

import furnace_b200 as fz
from tests.test_kvq8 import PAGE, Dev, gpu  # noqa: F401  (the module's GPU fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("long", [100, 400])
def test_idle_slots_of_a_uniform_batch(gpu, new, long):
    """A batch of fixed size without starts (a captured decode step): slots of
    length 0 have no rows.  Their output rows stay, no status is set, and the
    other sequences' results are as ever."""
    d = Dev(20, 8, 2, 64, 500)
    lens = [0, 50, 0, long, 0]
    t = d.table(lens)
    d.append(t, lens, lens)
    lens = [n and n + new for n in lens]
    n = 5 * new
    s = d.seqs(t, lens, [new] * 5, uniform=True)
    k, v, q = d.rows(n, 2, fz.F32), d.rows(n, 2, fz.F32), d.rows(n, 8, fz.F32)
    d.c.append(s, k[1].data_ptr(), v[1].data_ptr(), 128, stream=d.stream())
    d.c.status(d.stream())
    out = gpu.full((n, 512), 99.0, device="cuda")
    work = gpu.empty(d.c.attend_work(s), dtype=gpu.uint8, device="cuda")
    d.c.attend(s, q[1].data_ptr(), out.data_ptr(), 512, 512, work.data_ptr(), work.numel(), stream=d.stream())
    d.c.status(d.stream())
    back = gpu.full((2, n, 128), 7.0, device="cuda")
    d.c.read(s, back[0].data_ptr(), back[1].data_ptr(), 128, stream=d.stream())
    d.c.status(d.stream())
    got, back = out.view(n, 8, 64).cpu().numpy(), back.cpu().numpy()
    for i, length in enumerate(lens):
        r = slice(i * new, (i + 1) * new)
        if not length:
            assert (got[r] == 99.0).all() and (back[:, r] == 7.0).all()
            continue
        d.plain.append(t[i], length, k[0][r], v[0][r])
        want, tol = d.plain.attend(t[i], length, q[0][r])
        assert (np.abs(got[r] - want) <= tol).all()
        rows = np.stack(d.plain.rows(t[i], length - new, length, np.float32))
        assert np.array_equal(back[:, r], rows.transpose(0, 2, 1, 3).reshape(2, new, 128))
    d.check_cache([(t[i], length) for i, length in enumerate(lens) if length])


def test_a_uniform_sequence_shorter_than_its_rows_is_still_refused(gpu):
    d = Dev(8, 4, 2, 64, 200)
    t = d.table([40, 2])
    d.append(t, [40, 2], [40, 2])
    s = d.seqs(t, [40, 2], [3, 3], uniform=True)
    q, out = d.rows(6, 4, fz.F32), gpu.zeros(6, 256, device="cuda")
    work = gpu.empty(d.c.attend_work(s), dtype=gpu.uint8, device="cuda")
    d.c.attend(s, q[1].data_ptr(), out.data_ptr(), 256, 256, work.data_ptr(), work.numel(), stream=d.stream())
    with pytest.raises(fz.FurnaceError, match="lengths or rows"):
        d.c.status(d.stream())


def test_status_keeps_what_another_stream_finds_meanwhile(gpu):
    """A report takes the bits that it names and no others: one that a call on
    another stream sets while a report is under way is in this report or in the
    next.  The other stream's call is delayed by more and more, so that it meets
    every moment of the report."""
    d = Dev(8, 4, 2, 64, 200)
    t = d.table([40, 90])
    d.append(t, [40, 90], [40, 90])
    bad_len = d.seqs(t[:1], [PAGE * t.shape[1] + 1], [1])
    bad_page = d.seqs(np.full((1, 2), d.n_pages, np.int32), [90], [1])
    out = gpu.zeros(2, 1, 128, device="cuda")
    other = gpu.cuda.Stream()
    gpu.cuda.synchronize()

    def report(stream):
        try:
            d.c.status(stream)
            return ""
        except fz.FurnaceError as e:
            return str(e)

    for delay in range(0, 200000, 400):  # cycles
        d.c.read(bad_len, out[0].data_ptr(), None, 128, stream=d.stream())
        with gpu.cuda.stream(other):
            gpu.cuda._sleep(delay)
        d.c.read(bad_page, out[1].data_ptr(), None, 128, stream=other.cuda_stream)
        first = report(d.stream())
        second = report(other.cuda_stream)
        assert "lengths or rows" in first and "lengths or rows" not in second, (delay, first, second)
        assert ("page number" in first) != ("page number" in second), (delay, first, second)
    d.c.status(d.stream())
