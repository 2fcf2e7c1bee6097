"""The 8-bit paged KV cache's attention over long contexts, against a bound that
a page left out, or taken twice, does not pass.

The bound goes by what the kernels add up.  With p_t the weights, A = sum p_t
|v_t| of an output element and U = 2^-23 (one f32 operation that truncates):

  scores      off by d = (hd + 8) U sum |q_i k_i| and 4 U |score|; a weight by d
              and by 32 U more (the exponential's 2^-22, the logarithm of a value
              scale between 2^-8 and 2^8, at most 8 * 2^-22, the two fp16 parts)
  products    16 matrix instructions (128 positions, two parts) of 17 addends
              that truncate: 272 U of the step's sum of p_t |v_t|
  numerator   one rounded addition (U / 2) a page, 64 for the ends and joins
  denominator two additions a page, 64 for the ends and joins

so that an element is off by at most (2 d + 64 U + 272 U + (3 pages + 128) U / 2)
A: with queries of 2^-6, whose scores are small, 1e-4 of A at 30000 positions."""

import numpy as np
import pytest

import furnace_b200 as fz
from tests.test_kvq8 import BLOCK, PAGE, U, Dev, Plain, block_index, gpu, rope_table  # noqa: F401

SPREAD = 2.0 ** -6  # of the queries


def weights(plain, table, length, q, h, window=0, sinks=0):
    """Of one row (q [heads, hd], the sequence's last) and head: weights [length],
    values, the score error d."""
    group = q.shape[0] // plain.kv
    k, v = (x[h // group] for x in plain.rows(table, 0, length))
    qr = plain.rotate(q[None].astype(np.float64), np.array([length - 1]), np.float64)[0, h]
    s = k @ qr * plain.hd ** -0.5
    t = np.arange(length)
    seen = np.ones(length, bool) if not window else (t >= length - window) | (t < sinks)
    p = np.where(seen, np.exp(s - s[seen].max()), 0.0)
    d = (plain.hd + 8) * U * (np.abs(k) @ np.abs(qr)).max() * plain.hd ** -0.5 + 4 * U * np.abs(s).max()
    return p / p.sum(), v, d


def result_and_bound(p, v, d):
    pages = (np.count_nonzero(p) + PAGE - 1) // PAGE + 2
    eps = 2 * d + (64 + 272 + (3 * pages + 128) / 2) * U
    return p @ v, eps * (p @ np.abs(v)) + 1e-40


def fill(plain, rng, pages):
    """Random codes and scales in `pages` of a restatement; returns them as the device holds them."""
    kv, hd = plain.kv, plain.hd
    raw = rng.integers(1, 256, (len(pages), kv, 2, PAGE // BLOCK, BLOCK * hd), dtype=np.uint8)
    scales = ((rng.random((len(pages), kv, 2, PAGE // BLOCK)) + 0.5) / 52).astype(np.float32)
    for w, at in enumerate(block_index(hd)):
        plain.codes[pages, :, w] = raw[:, :, w][..., at].astype(np.int32) - 128
    plain.scales[pages] = scales
    return raw, scales


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("length, window", [(8000, 0), (20000, 0), (32768, 0), (20000, 9000)])
def test_the_bound_sees_every_page(hd, length, window):
    """Whichever page, or half of one (what a warp takes), is left out or taken
    twice: the result moves by more than the bound, with a fifth to spare."""
    rng = np.random.default_rng(length + hd)
    n = (length + PAGE - 1) // PAGE
    plain = Plain(n, 1, hd, rope_table(length, hd))
    table = rng.permutation(n)
    fill(plain, rng, np.arange(n))
    q = (rng.standard_normal((4, hd)) * SPREAD).astype(np.float32)
    ratio = 0.0
    for h in range(4):
        p, v, d = weights(plain, table, length, q, h, window)
        out, tol = result_and_bound(p, v, d)
        lo = max(0, length - window) if window else 0
        first, last = -(-lo // 32), length // 32  # whole halves of pages in sight
        share = p[first * 32:last * 32].reshape(-1, 32)
        part = np.einsum("nt,ntd->nd", share, v[first * 32:last * 32].reshape(-1, 32, hd))
        share = share.sum(1)
        gone = (out - part) / (1 - share)[:, None]
        twice = (out + part) / (1 + share)[:, None]
        ratio = np.maximum(ratio, np.minimum(np.abs(gone - out), np.abs(twice - out)) / tol)
    assert ratio.max(-1).min() > 1.2, ratio.max(-1).min()


def filled(lens, heads, kv, hd, seed=0):
    d = Dev(sum((n + PAGE - 1) // PAGE for n in lens), heads, kv, hd, max(lens), seed)
    t = d.table(lens)
    raw, scales = fill(d.plain, d.rng, np.arange(d.n_pages))
    d.codes.copy_(d.t.from_numpy(raw.reshape(d.codes.shape)))
    d.scales.copy_(d.t.from_numpy(scales))
    return d, t


def check(d, t, lens, news, rows, heads, dtype=fz.F32, window=0, sinks=0):
    q = d.rows(int(sum(news)), d.heads, dtype, spread=SPREAD)
    _, got = d.attend(t, lens, news, dtype, q=q, window=window, sinks=sinks)
    r = 0
    for i, (length, new) in enumerate(zip(lens, news)):
        for j in sorted({x % new for x in rows}):
            for h in heads:
                p, v, e = weights(d.plain, t[i], length - new + j + 1, q[0][r + j], h, window, sinks)
                want, tol = result_and_bound(p, v, e)
                if dtype == fz.F16:
                    tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
                err = np.abs(got[r + j, h] - want)
                assert (err <= tol).all(), (i, j, h, float((err / tol).max()))
        r += new
    d.c.status(d.stream())


@pytest.mark.gpu
@pytest.mark.parametrize("hd, kv, group, dtype", [(128, 2, 7, fz.F32), (64, 4, 2, fz.F16)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (9000, 70)])
def test_tokens_over_long_contexts(gpu, hd, kv, group, dtype, window, sinks):
    """Runs of many pages that end inside sequences and span several."""
    lens = [20000, 1, 640, 16001, 700, 18000, 64, 65, 9000, 32768, 8000, 5555]
    d, t = filled(lens, kv * group, kv, hd)
    heads = (0, group, kv * group - 1)
    check(d, t, lens, [1] * len(lens), (0,), heads, dtype, window, sinks)
    few = [min(3, n) for n in lens]
    check(d, t, lens, few, (0, -1), heads[::2], dtype, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("hd, kv, group, dtype", [(128, 1, 7, fz.F32), (64, 2, 4, fz.F16)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (9000, 5)])
def test_prompt_pieces_over_long_contexts(gpu, hd, kv, group, dtype, window, sinks):
    """Parts of many pages, in one sequence and in two."""
    lens = [20100, 8050]
    d, t = filled(lens, kv * group, kv, hd, seed=1)
    heads = (0, kv * group - 1)
    check(d, t[:1], lens[:1], [300], (0, 130, -1), heads, dtype, window, sinks)
    check(d, t, lens, [700, 260], (0, 130, -1), heads, dtype, window, sinks)
