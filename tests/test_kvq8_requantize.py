"""What a cached row may be off by after its block was filled a few positions at
a time: half a code when it is appended, and up to half a code more for every
later call that raises the block's scale (include/furnace.h)."""

import numpy as np
import pytest

import furnace_b200 as fz
from tests.test_kvq8 import BLOCK, Dev, Plain, gpu  # noqa: F401


def drift(kv, hd):
    """Values of one block, a position a call: each call's largest raises the
    scale by just so much that codes near 100 of the rows before round up again."""
    x = np.full((BLOCK, kv, hd), 0.1, np.float32)
    grow = np.float64(100.0) / 99.51
    for p in range(BLOCK):
        x[p, :, 0] = 127.0 * grow ** p
        x[p, :, 1] = 100.0
    x[0, :, 2:] = np.linspace(-127, 127, hd - 2)
    return x


def noise(rng, kv, hd):
    return (rng.standard_normal((BLOCK, kv, hd)) * np.exp(rng.uniform(-2, 2, (BLOCK, 1, 1)))).astype(np.float32)


def bound(x, pieces):
    """Per position: codes of the block's last scale.  A code's own f32 rounding
    is 127 * 2^-23 of one at most, a recode's the same."""
    ends = np.cumsum(pieces)
    tops = [np.abs(x[:e]).max((0, 2)) for e in ends]  # [kv]
    out = np.zeros(x.shape[:2])
    for i, (e, n) in enumerate(zip(ends, pieces)):
        raised = sum((tops[j] > tops[j - 1]).astype(int) for j in range(i + 1, len(ends))) if i + 1 < len(ends) else 0
        out[e - n:e] = (1 + raised) * (0.5 + 127 * 2.0 ** -22)
    return out * (tops[-1] / 127)


PIECES = [[1] * 16, [16], [5, 1, 1, 6, 3], [15, 1], [1, 15]]


@pytest.mark.parametrize("pieces", PIECES, ids=str)
def test_rows_stay_within_half_a_code_a_raise(pieces):
    rng = np.random.default_rng(0)
    worst = 0.0
    for x in [drift(2, 64)] + [noise(rng, 2, 64) for _ in range(20)]:
        plain = Plain(1, 2, 64, None)
        at = 0
        for n in pieces:
            plain.append([0], at + n, x[at:at + n], x[at:at + n])
            at += n
        limit = bound(x, pieces)
        for rows in plain.rows([0], 0, BLOCK):
            off = np.abs(rows.transpose(1, 0, 2) - x)
            assert (off.max(2) <= limit).all()
            worst = max(worst, (off / (np.abs(x).max((0, 2)) / 127)[None, :, None]).max())
    if pieces == [1] * 16:
        assert worst > 6  # the bound of 8 codes is nearly reached: it says no more than what can happen


@pytest.mark.gpu
@pytest.mark.parametrize("pieces", PIECES, ids=str)
@pytest.mark.parametrize("hd", [64, 128])
def test_the_device_does_the_same(gpu, hd, pieces):
    rng = np.random.default_rng(1)
    for x in (drift(2, hd), noise(rng, 2, hd)):
        d = Dev(1, 2, 2, hd)
        t, at = d.table([BLOCK]), 0
        for n in pieces:
            rows = (x[at:at + n], gpu.from_numpy(x[at:at + n].reshape(n, -1)).cuda())
            at += n
            d.append(t, [at], [n], k=rows, v=rows)
        gpu.cuda.synchronize()
        d.check_cache([(t[0], BLOCK)])
        back = gpu.zeros(2, BLOCK, 2 * hd, device="cuda")
        s = d.seqs(t, [BLOCK], [BLOCK])
        d.c.read(s, back[0].data_ptr(), back[1].data_ptr(), 2 * hd, stream=d.stream())
        off = np.abs(back.view(2, BLOCK, 2, hd).cpu().numpy() - x)
        assert (off.max(3) <= bound(x, pieces)).all()
        d.c.status(d.stream())
