"""The 8-bit paged KV cache's attention in the forms that sizes select: long
prompts cut into parts, hundreds of sequences, many tiles for one run, a whole
short sequence at once; and what surrounds a call: its workspace's ends,
captured graphs, shared pages."""

import numpy as np
import pytest

import furnace_b200 as fz
from tests.test_kvq8 import PAGE, Dev, gpu  # noqa: F401  (the module's GPU fixture)

pytestmark = pytest.mark.gpu


def _sampled_rows(d, table, lens, news, rows, dtype=fz.F32, **kw):
    """check_attend for a few rows of a long call only (the restatement is slow)."""
    q, got = d.attend(table, lens, news, dtype, **kw)
    kw = {k: v for k, v in kw.items() if k in ("window", "sinks", "scale")}
    r = 0
    for i, (length, new) in enumerate(zip(lens, news)):
        for j in sorted({x % new for x in rows}) if new else []:
            pos = length - new + j + 1
            want, tol = d.plain.attend(table[i], pos, q[r + j:r + j + 1], **kw)
            if dtype == fz.F16:
                tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
            err = np.abs(got[r + j:r + j + 1] - want)
            assert (err <= tol).all(), (i, j, float((err / tol).max()), float(err.max()))
        r += new
    d.c.status(d.stream())


@pytest.mark.parametrize("hd, kv, group, dtype", [(128, 1, 7, fz.F32), (64, 2, 4, fz.F16), (128, 2, 1, fz.F16),
                                                  (64, 1, 16, fz.F32)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (700, 5), (64, 0)])
def test_prompt_pieces_behind_long_prefixes(gpu, hd, kv, group, dtype, window, sinks):
    """One sequence, few tiles of rows: the pages are cut into parts (an odd
    number of them, parts without a page that a row sees)."""
    d = Dev(120, kv * group, kv, hd, 7000)
    lens = [3335, 2100]
    t = d.table(lens)
    d.append(t, lens, lens)
    for i, news in ((0, [300]), (0, [1100]), (1, [2100])):
        _sampled_rows(d, t[i:i + 1], lens[i:i + 1], news, (0, 1, 63, 64, 127, 128, 777, -1), dtype, window=window,
                      sinks=sinks)
    _sampled_rows(d, t, lens, [257, 640], (0, 200, -1), dtype, window=window, sinks=sinks)


def test_long_prompt_with_scales_far_apart_and_any_softmax_scale(gpu):
    d = Dev(40, 8, 1, 128)
    lens = [2000]
    t = d.table(lens)
    at = 0
    for b in range(10):
        k = d.rows(200, 1, fz.F32, spread=[1.0, 4.0, 0.01][b % 3])
        v = d.rows(200, 1, fz.F32, spread=10.0 ** (b - 5))
        at += 200
        d.append(t, [at], [200], k=k, v=v)
    for scale in (None, -0.03, 0.5):
        kw = {} if scale is None else {"scale": scale}
        _sampled_rows(d, t, lens, [900], (0, 1, 130, 500, -1), **kw)
        _sampled_rows(d, t, lens, [2], (0, 1), **kw)
    for spread in (1e-25, 1e30):
        e = Dev(40, 8, 1, 64, 2100)
        t = e.table([2000])
        e.append(t, [2000], [2000], v=e.rows(2000, 1, fz.F32, spread=spread))
        _sampled_rows(e, t, [2000], [800], (0, 400, -1))


def test_hundreds_of_sequences(gpu):
    """More sequences than a CTA has threads, ragged, some empty, some longer
    than the form for short ones takes."""
    rng = np.random.default_rng(1)
    lens = [int(x) for x in rng.integers(0, 90, 300)]
    lens[150], lens[299], lens[0] = 700, 300, 0
    d = Dev(sum((n + PAGE - 1) // PAGE for n in lens), 12, 2, 64, 800)
    t = d.table(lens)
    d.append(t, lens, lens)
    news = [min(1, n) for n in lens]
    d.check_attend(t, lens, news)
    d.check_attend(t, lens, [min(3, n) for n in lens], window=40, sinks=3)
    short = [min(n, 250) for n in lens]
    d.check_attend(np.ascontiguousarray(t[:, :4]), short, [min(1, n) for n in short], fz.F16)


def test_many_tiles_for_every_run(gpu):
    """Runs of dozens of pages that end inside sequences and span several."""
    d = Dev(1400, 16, 8, 128, 20000)
    lens = [20000, 1, 640, 16001, 700, 18000, 64, 65, 9000, 4000, 8000, 5555]
    t = d.table(lens)
    rows = sum(lens)
    k = d.rows(rows, 8, fz.F16)
    d.append(t, lens, lens, fz.F16, k=k, v=k)
    d.check_attend(t, lens, [1] * len(lens), uniform=True)


@pytest.mark.parametrize("news, lens", [([1], [600]), ([3], [200]), ([900], [1800])])
def test_workspace_ends(gpu, news, lens):
    """Exactly attend_work bytes are enough, and nothing past them is written."""
    d = Dev(32, 14, 2, 128, 2000)
    t = d.table(lens)
    d.append(t, lens, lens)
    s = d.seqs(t, lens, news)
    n = d.c.attend_work(s)
    work = gpu.full((n + 4096,), 0xA5, dtype=gpu.uint8, device="cuda")
    q, out = d.rows(sum(news), 14, fz.F32), gpu.zeros(sum(news), 14 * 128, device="cuda")
    d.c.attend(s, q[1].data_ptr(), out.data_ptr(), 1792, 1792, work.data_ptr(), n, stream=d.stream())
    gpu.cuda.synchronize()
    assert (work[n:] == 0xA5).all()
    with pytest.raises(fz.FurnaceError, match="work"):
        d.c.attend(s, q[1].data_ptr(), out.data_ptr(), 1792, 1792, work.data_ptr(), n - 1, stream=d.stream())


def test_two_captured_graphs_replayed_together(gpu):
    """A prompt piece and a decode step, each captured with its own workspace,
    replayed at the same time on two streams over the same cache, again and
    again, give what they give alone."""
    d = Dev(100, 14, 2, 128, 3000)
    lens = [2500, 1800]
    t = d.table(lens)
    d.append(t, lens, lens)
    graphs = []
    for news in ([600, 500], [1, 1]):
        s, n = d.seqs(t, lens, news), sum(news)
        q, out = d.rows(n, 14, fz.F32), gpu.zeros(n, 1792, device="cuda")
        work = gpu.empty(d.c.attend_work(s), dtype=gpu.uint8, device="cuda")
        side, g = gpu.cuda.Stream(), gpu.cuda.CUDAGraph()
        side.wait_stream(gpu.cuda.current_stream())
        with gpu.cuda.graph(g, stream=side):
            d.c.attend(s, q[1].data_ptr(), out.data_ptr(), 1792, 1792, work.data_ptr(), work.numel(),
                       stream=gpu.cuda.current_stream().cuda_stream)
        g.replay()
        gpu.cuda.synchronize()
        graphs.append((g, side, out, out.clone(), s, q, work))
        assert out.abs().sum() > 0
    for _ in range(20):
        for g, side, out, *_ in graphs:
            with gpu.cuda.stream(side):
                out.zero_()
                g.replay()
    gpu.cuda.synchronize()
    for g, side, out, want, *_ in graphs:
        assert gpu.equal(out, want)
    d.c.status(d.stream())


def test_pages_shared_between_sequences(gpu):
    """Two sequences that start with the same pages (a prompt kept once), and
    the same sequence twice in a call."""
    d = Dev(20, 8, 2, 64, 800)
    base = d.table([640])
    d.append(base, [640], [640])
    own = d.table([100])  # pages for the second sequence's own end
    two = np.full((3, 12), -7, np.int32)
    two[0, :10] = two[1, :10] = two[2, :10] = base[0, :10]
    two[1, 10:12] = own[0, :2]
    d.append(two[1:2], [700], [60])
    d.check_attend(two, [640, 700, 640], [1, 2, 1])


def test_rows_of_a_fused_projection(gpu):
    """q, k and v as columns of one row, the result into columns of another,
    for a prompt and for one token."""
    d = Dev(30, 8, 2, 64, 1500)
    lens, width = [1400], (8 + 2 + 2) * 64
    t = d.table(lens)
    d.append(t, [200], [200])
    for new, end in ((1100, 1300), (1, 1301)):
        x = d.rng.standard_normal((new, 12, 64)).astype(np.float32)
        qkv = gpu.from_numpy(x.reshape(new, -1)).cuda()
        out = gpu.full((new, 640), 5.0, device="cuda")
        s = d.seqs(t, [end], [new])
        work = gpu.empty(d.c.attend_work(s), dtype=gpu.uint8, device="cuda")
        d.c.append(s, qkv.data_ptr() + 4 * 512, qkv.data_ptr() + 4 * 640, width, stream=d.stream())
        d.c.attend(s, qkv.data_ptr(), out.data_ptr() + 4 * 64, width, 640, work.data_ptr(), work.numel(),
                   stream=d.stream())
        gpu.cuda.synchronize()
        d.plain.append(t[0], end, x[:, 8:10], x[:, 10:12])
        d.check_cache([(t[0], end)])
        got = out.cpu().numpy()
        assert (got[:, :64] == 5.0).all() and (got[:, 576:] == 5.0).all()
        for j in (0, new // 2, new - 1):
            want, tol = d.plain.attend(t[0], end - new + j + 1, x[j:j + 1, :8])
            assert (np.abs(got[j, 64:576].reshape(1, 8, 64) - want) <= tol).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_codes_at_rounding_borders(gpu, hd):
    """Values a few units in the last place around half codes, for scales of
    every magnitude (smallest 2^-140, largest 2^120): the codes are those of a
    rounded f32 division, bit for bit."""
    n = 16 * 44
    d = Dev((n + PAGE - 1) // PAGE, 2, 2, hd)
    t = d.table([n])
    shape = (44, 16, 2, hd)
    exps = np.linspace(-140, 120, 44).astype(int)
    both = []
    for _ in range(2):
        top = (np.ldexp(d.rng.uniform(1, 2, (44, 1, 2, 1)), exps[:, None, None, None]) * 63.5).astype(np.float32)
        scale = top / np.float32(127)
        x = ((d.rng.integers(-127, 127, shape) + 0.5).astype(np.float32) * scale).astype(np.float32)
        x = (x.view(np.int32) + d.rng.integers(-3, 4, shape).astype(np.int32)).view(np.float32)
        x = np.clip(np.where(np.isfinite(x), x, np.float32(0)), -top, top)
        x[:, 0, :, 0] = top[:, 0, :, 0]
        x = x.reshape(n, 2, hd)
        both.append((x, gpu.from_numpy(x.reshape(n, -1)).cuda()))
    d.append(t, [n], [n], k=both[0], v=both[1])
    gpu.cuda.synchronize()
    d.check_cache([(t[0], n)])
    d.c.status(d.stream())


@pytest.mark.parametrize("hd, kv, dtype", [(64, 16, fz.F16), (128, 8, fz.F32), (128, 7, fz.F16), (64, 9, fz.F32)])
def test_append_of_more_blocks_than_fit_at_once(gpu, hd, kv, dtype):
    """One sequence, so many blocks and heads that a CTA takes several of them,
    entered in the middle of a block; what is read back is what was written."""
    end = 3701
    d = Dev((end + PAGE - 1) // PAGE, kv, kv, hd, end)
    t = d.table([end])
    d.append(t, [37], [37], dtype)
    d.append(t, [end], [end - 37], dtype, k=d.rows(end - 37, kv, dtype, spread=3.0))
    gpu.cuda.synchronize()
    d.check_cache([(t[0], end)])
    s = d.seqs(t, [end], [end])
    k, v = (gpu.full((end, kv * hd), 9.0, device="cuda") for _ in range(2))
    d.c.read(s, k.data_ptr(), v.data_ptr(), kv * hd, stream=d.stream())
    gpu.cuda.synchronize()
    for got, want in zip((k, v), d.plain.rows(t[0], 0, end, np.float32)):
        assert np.array_equal(got.cpu().numpy().reshape(end, kv, hd).transpose(1, 0, 2), want)
    d.c.status(d.stream())
