"""Calls around the edges of the 8-bit paged KV cache."""

import math

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


def _no_numbers(d, table, lens, news, q, bad, window=0, sinks=0):
    """Attention where the key blocks of positions `bad` are NaN: rows that see
    one are NaN, the others what they are without."""
    q, got = d.attend(table, lens, news, q=q, **(dict(window=window, sinks=sinks) if window else {}))
    n, new = lens[0], news[0]
    pos = np.arange(n - new, n)
    seen = np.arange(n)[None] <= pos[:, None]
    if window:
        seen &= (np.arange(n)[None] > pos[:, None] - window) | (np.arange(n)[None] < sinks)
    hit = (seen & bad[None, :n]).any(-1) | np.isnan(q).any((1, 2))
    assert np.isnan(got[hit]).all(), np.argwhere(~np.isnan(got[hit]).all((1, 2)))[:4]
    for j in np.flatnonzero(~hit)[:: max(1, (~hit).sum() // 6)]:
        want, tol = d.plain.attend(table[0], int(pos[j]) + 1, q[j:j + 1], window=window, sinks=sinks)
        assert (np.abs(got[j] - want[0]) <= tol[0]).all(), j
    return hit


@pytest.mark.parametrize("new", [1, 3, 150, 900])
@pytest.mark.parametrize("span", [(0, 16), (0, 640), (640, 1296), (1100, 1300)])
def test_keys_that_are_no_numbers_reach_every_row_that_sees_them(gpu, new, span):
    """In every form of the attention (single tokens, a few, prompts whose pages
    are cut into parts), also where all that a row or a part sees is NaN: never
    a result that leaves those positions out."""
    d = Dev(24, 8, 2, 64, 1400)
    n = 1300
    t = d.table([n])
    d.append(t, [n], [n])
    blocks = np.arange(n) // 16
    bad = (blocks >= span[0] // 16) & (blocks <= (span[1] - 1) // 16)
    for b in np.unique(blocks[bad]):
        d.scales[int(t[0, b // 4]) + d.first, :, 0, b % 4] = math.nan
    q = d.rows(new, 8, fz.F32)
    hit = _no_numbers(d, t, [n], [new], q, bad)
    assert hit.all() or new == 900
    _no_numbers(d, t, [n], [new], q, bad, window=90, sinks=3)
    _no_numbers(d, t, [n], [new], q, bad, window=200)
    short = min(new, 40)
    _no_numbers(d, t[:, :1], [40], [short], d.rows(short, 8, fz.F32), bad)


@pytest.mark.parametrize("new", [2, 150, 900])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_queries_that_are_no_numbers_give_none(gpu, new, value):
    """A query with a NaN or an infinity has no softmax; the rows beside it are
    as ever."""
    d = Dev(24, 8, 2, 64, 1400)
    t = d.table([1300])
    d.append(t, [1300], [1300])
    x, dev = d.rows(new, 8, fz.F32)
    at = [0, new // 2, new - 1] if new > 2 else [1]
    for j in at:
        x[j] = math.nan  # what the check takes such a row for
        dev[j, 5::64] = value
    _no_numbers(d, t, [1300], [new], (x, dev), np.zeros(1300, bool))
    _no_numbers(d, t, [1300], [new], (x, dev), np.zeros(1300, bool), window=100, sinks=2)


@pytest.mark.parametrize("new", [1, 5, 33, 130, 900])
@pytest.mark.parametrize("spread", [3e33, 6e37])
def test_values_up_to_the_end_of_the_range(gpu, new, spread):
    """Values whose scales are far above 2^96, with scores that differ by many
    powers of two: every form keeps the small weights, and nothing overflows
    that the result does not."""
    d = Dev(24, 8, 2, 64, 1400)
    n = 1300
    t = d.table([n])
    k, v = d.rows(n, 2, fz.F32, spread=3.0), d.rows(n, 2, fz.F32)
    v[0][:] = np.clip(v[0], -4, 4) * np.float32(spread)
    v[1][:] = gpu.from_numpy(v[0].reshape(n, -1)).cuda()
    d.append(t, [n], [n], k=k, v=v)
    for kw in ({}, dict(window=300, sinks=5)):
        d.check_attend(t, [n], [new], **kw)
    short = min(new, 60)
    d.check_attend(t[:, :1], [60], [short])


@pytest.mark.parametrize("new", [1, 5, 130, 900])
def test_value_scales_80_powers_of_two_apart(gpu, new):
    """Blocks of tiny values between blocks of huge ones: their weights count in
    the denominator all the same."""
    d = Dev(24, 8, 2, 64, 1400)
    n = 1280
    t = d.table([n])
    k, v = d.rows(n, 2, fz.F32, spread=2.0), d.rows(n, 2, fz.F32)
    v[0][:] *= np.repeat(np.where(np.arange(n // 16) % 3 == 0, 2.0 ** 90, 2.0 ** 10), 16)[:, None, None].astype(np.float32)
    v[1][:] = gpu.from_numpy(v[0].reshape(n, -1)).cuda()
    d.append(t, [n], [n], k=k, v=v)
    d.check_attend(t, [n], [new])
    d.check_attend(t, [n], [new], window=200, sinks=20)


@pytest.mark.parametrize("new", [1, 150, 900])
@pytest.mark.parametrize("block", [0, 1, 34, 35, 81])
def test_value_scales_that_are_no_numbers(gpu, new, block):
    """One block of values without numbers, next to one with: the rows that see
    it are NaN, the others as ever."""
    d = Dev(24, 8, 2, 64, 1400)
    n = 1300
    t = d.table([n])
    d.append(t, [n], [n])
    d.scales[int(t[0, block // 4]) + d.first, :, 1, block % 4] = math.nan
    bad = np.arange(n) // 16 == block
    q = d.rows(new, 8, fz.F32)
    _no_numbers(d, t, [n], [new], q, bad)
    _no_numbers(d, t, [n], [new], q, bad, window=100, sinks=3)


@pytest.mark.parametrize("new", [1, 130, 900])
@pytest.mark.parametrize("spread", [1e-29, 1e-33, 0.0])
def test_tiny_and_zero_values_over_many_positions(gpu, new, spread):
    """Scales down to 2^-96 keep f32's precision; below that the two fp16 parts of
    a weight, at most 1, end at 2^-36, and zeros stay zeros."""
    d = Dev(24, 8, 2, 64, 1400)
    n = 1300
    t = d.table([n])
    d.append(t, [n], [n], v=d.rows(n, 2, fz.F32, spread=spread))
    q, got = d.attend(t, [n], [new])
    want, tol = d.plain.attend(t[0], n, q)
    # n weights off by half of 2^-35, codes up to 127, a denominator of 1 or more
    assert (np.abs(got - want) <= tol + n * 127 * 2.0 ** -36 * 2.0 ** -96).all()
    assert spread or not got.any()


@pytest.mark.parametrize("hd, kv, group, dtype", [(128, 2, 7, fz.F32), (64, 1, 4, fz.F16)])
def test_one_prompt_beside_single_tokens(gpu, hd, kv, group, dtype):
    """What a serving step looks like: a prompt among sequences with a token
    each, and idle ones; its rows, theirs and the cache are as in calls of their
    own."""
    lens = [700, 40, 0, 1033, 64, 1, 300, 0, 129]
    d = Dev(60, kv * group, kv, hd, 1100)
    t = d.table(lens)
    news = [1, 1, 0, 1033, 1, 1, 1, 0, 1]
    old = [n - new for n, new in zip(lens, news)]
    d.append(t, old, old, dtype)
    d.append(t, lens, news, dtype)
    gpu.cuda.synchronize()
    d.check_cache([(t[i], n) for i, n in enumerate(lens) if n])
    d.check_attend(t, lens, news, dtype)
    d.check_attend(t, lens, news, dtype, window=100, sinks=5)


@pytest.mark.parametrize("new", [1, 12, 130])
def test_a_table_much_wider_than_its_sequences(gpu, new):
    """A table as wide as the longest sequence a server takes, and short
    sequences: the entries past their ends are not read."""
    lens = [130, 140, 1, 400]
    d = Dev(20, 8, 2, 64, 500)
    t = d.table(lens, spare=505)
    d.append(t, lens, lens)
    news = [min(new, n) for n in lens]
    d.check_attend(t, lens, news)
    d.check_attend(t, lens, news, window=70, sinks=2)
