"""Addresses that a kernel could not read: refused before any device work."""

import pytest

import furnace_b200 as fz
from tests.test_kvq8 import FAKE, _cache, _seqs


@pytest.mark.parametrize("cache, seqs, words", [
    (dict(status=FAKE + 2), {}, "status"),
    ({}, dict(pages=FAKE + 1), "page table"),
    ({}, dict(lens=FAKE + 2), "lengths"),
    ({}, dict(starts=FAKE + 3), "row starts"),
])
def test_words_off_their_boundary_are_refused(cache, seqs, words):
    c, s = _cache(**cache), _seqs(**seqs)
    calls = [lambda: c.append(s, FAKE, FAKE, 128), lambda: c.read(s, FAKE, FAKE, 128), lambda: c.attend_work(s),
             lambda: c.attend(s, FAKE, FAKE + (1 << 16), 512, 512, FAKE, 1 << 30)]
    if cache:
        calls.append(c.status)
    for call in calls:
        with pytest.raises(fz.FurnaceError, match=words) as e:
            call()
        assert e.value.code == fz.FZ_EINVAL and "4-byte" in str(e.value)
