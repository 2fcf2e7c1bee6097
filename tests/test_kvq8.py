"""The 8-bit paged KV cache (fz_kvq8_*): append with rotation, attention with
and without a sliding window, read-back.

`Plain` restates the append in numpy f32 (the same elementary operations, so
codes and scales must be equal bit for bit) and the attention in 64 bits over
what the cache stands for.
"""

import ctypes as C
import math

import numpy as np
import pytest

import furnace_b200 as fz

PAGE, BLOCK = fz.KVQ8_PAGE, fz.KVQ8_BLOCK
U = 2.0 ** -23  # unit of one f32 operation, truncating accumulation allowed


def k_at(p, d, hd):
    return (p // 8) * 8 * hd + (d // 64) * 512 + (p % 8) * 64 + d % 64


def v_at(p, d):
    return (d // 32) * 512 + (d % 8) * 64 + (p % 8 // 2) * 16 + (d % 32 // 8) * 4 + (p // 8) * 2 + p % 2


def block_index(hd):
    p, d = np.meshgrid(np.arange(BLOCK), np.arange(hd), indexing="ij")
    return k_at(p, d, hd), v_at(p, d)


def rope_table(n, hd, theta=1e6):
    a = np.arange(n, dtype=np.float64)[:, None] * theta ** (-2.0 * np.arange(hd // 2) / hd)[None]
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


class Plain:
    """codes [page, kv, 2, block, 16, hd] as values, scales [page, kv, 2, block]."""

    def __init__(self, n_pages, kv, hd, rope):
        self.kv, self.hd, self.rope = kv, hd, rope
        self.codes = np.zeros((n_pages, kv, 2, PAGE // BLOCK, BLOCK, hd), np.int32)
        self.scales = np.zeros((n_pages, kv, 2, PAGE // BLOCK), np.float32)

    def rotate(self, x, pos, dtype=np.float32):
        """x [rows, heads, hd] at positions pos."""
        if self.rope is None:
            return x.astype(dtype)
        x, f = x.astype(dtype), self.rope[pos].astype(dtype)
        h = self.hd // 2
        a, b, c, s = x[..., :h], x[..., h:], f[:, None, :, 0], f[:, None, :, 1]
        return np.concatenate([a * c - b * s, a * s + b * c], -1)

    def append(self, table, length, k, v):
        """k, v [rows, kv, hd]: the last positions of a sequence of `length`."""
        new, old = k.shape[0], length - k.shape[0]
        x = np.stack([self.rotate(k, np.arange(old, length)), v.astype(np.float32)], 1)  # [rows, 2, kv, hd]
        for b in range(old // BLOCK, (length + BLOCK - 1) // BLOCK):
            lo, hi = max(old, b * BLOCK), min(length, (b + 1) * BLOCK)
            if hi <= lo:
                continue
            page, sub = table[b * BLOCK // PAGE], b % (PAGE // BLOCK)
            for w in range(2):
                for h in range(self.kv):
                    rows = x[lo - old:hi - old, w, h]
                    before = self.scales[page, h, w, sub]
                    scale = np.float32(np.abs(rows).max()) / np.float32(127)
                    kept = lo - b * BLOCK
                    codes = self.codes[page, h, w, sub]
                    if kept:
                        scale = max(scale, before)
                        if scale > before:
                            codes[:kept] = np.rint(codes[:kept].astype(np.float32) * (before / scale))
                    codes[kept:hi - b * BLOCK] = np.clip(np.rint(rows / scale), -127, 127) if scale > 0 else 0
                    self.scales[page, h, w, sub] = scale

    def rows(self, table, lo, hi, dtype=np.float64):
        """K and V [kv, hi - lo, hd] as the cache holds them."""
        p = np.arange(lo, hi)
        page, sub, tok = np.asarray(table)[p // PAGE], p // BLOCK % (PAGE // BLOCK), p % BLOCK
        c = self.codes[page, :, :, sub, tok].astype(dtype) * self.scales[page, :, :, sub][..., None].astype(dtype)
        return c[:, :, 0].transpose(1, 0, 2), c[:, :, 1].transpose(1, 0, 2)

    def attend(self, table, length, q, window=0, sinks=0, scale=None):
        """q [rows, heads, hd] -> (out, bound of |f32 result - out|)."""
        n, heads = q.shape[:2]
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        if n == 0 or length == 0:
            return out, tol
        k, v = self.rows(table, 0, length)
        scale = self.hd ** -0.5 if scale is None else scale
        pos = np.arange(length - n, length)
        qr = self.rotate(q.astype(np.float64), pos, np.float64)
        t = np.arange(length)
        for h in range(heads):
            kh, vh = k[h // (heads // self.kv)], v[h // (heads // self.kv)]
            s = qr[:, h] @ kh.T * scale
            seen = t[None] <= pos[:, None]
            if window:
                seen &= (t[None] > pos[:, None] - window) | (t[None] < sinks)
            s = np.where(seen, s, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[:, h] = p @ vh
            # |score error| <= (terms + a few roundings) x unit x sum of magnitudes (q's rotation and the split into
            # two 11-bit parts add under 8 units); a weight is off by that and the exponent's rounding (|s| units,
            # in base 2); numerator and denominator each add one unit per visible position
            mag = (np.abs(qr[:, h]) @ np.abs(kh).T * abs(scale)).max(-1)
            eps = ((self.hd + 8) * mag + 2 * np.abs(s[seen]).max() + 2 * seen.sum(-1) + 16) * U
            tol[:, h] = (2 * eps * np.abs(vh).max())[:, None] + 1e-40
        return out, tol


# ---------------------------------------------------------------------------
# Without a GPU: layout and refusals
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [64, 128])
def test_block_layout_is_a_bijection(hd):
    for at in block_index(hd):
        assert sorted(at.reshape(-1).tolist()) == list(range(BLOCK * hd))


FAKE = 1 << 20  # an address that no refused call may touch


def _cache(**over):
    a = dict(codes=FAKE, scales=FAKE, status=FAKE, n_pages=4, n_heads=8, n_kv_heads=2, head_dim=64, rope=FAKE,
             n_rope=256)
    a.update(over)
    return fz.KvQ8(**a)


def _seqs(**over):
    a = dict(pages=FAKE, lens=FAKE, n_seqs=2, max_pages=2, n_rows=8, starts=FAKE, max_new=4)
    a.update(over)
    return fz.KvQ8Seqs(**a)


@pytest.mark.parametrize("cache, seqs, args, words", [
    (dict(codes=None), {}, {}, "null cache buffer"),
    (dict(status=None), {}, {}, "null cache buffer"),
    (dict(codes=FAKE + 8), {}, {}, "16-byte"),
    (dict(rope=FAKE + 4), {}, {}, "16-byte"),
    (dict(head_dim=96), {}, {}, "head_dim 96"),
    (dict(head_dim=0), {}, {}, "head_dim 0"),
    (dict(n_kv_heads=0), {}, {}, "KV heads"),
    (dict(n_heads=7), {}, {}, "not divisible"),
    (dict(n_pages=0), {}, {}, "pages"),
    (dict(n_pages=1 << 31), {}, {}, "pages"),
    (dict(rope=None), {}, {}, "rotation table"),
    (dict(n_rope=0), {}, {}, "rotation table"),
    ({}, dict(pages=None), {}, "page table"),
    ({}, dict(lens=None), {}, "lengths"),
    ({}, dict(max_pages=0), {}, "pages per sequence"),
    ({}, dict(max_pages=1 << 26), {}, "pages per sequence"),
    ({}, dict(max_new=0), {}, "new positions"),
    ({}, dict(max_new=129), {}, "new positions"),
    ({}, dict(n_seqs=65536), {}, "sequences"),
    ({}, dict(n_rows=1 << 31), {}, "rows"),
    ({}, dict(starts=None, n_rows=7), {}, "rows for 2 sequences"),
    ({}, {}, dict(dtype=fz.Q8_0), "type 8"),
    ({}, {}, dict(ld=120), "row stride"),
    ({}, {}, dict(ld=130), "16-byte"),
    ({}, {}, dict(x=FAKE + 4), "16-byte"),
    ({}, {}, dict(x=None), "null"),
])
def test_refusals_before_any_device_work(cache, seqs, args, words):
    a = dict(x=FAKE, ld=128, dtype=fz.F32)
    a.update(args)
    c, s = _cache(**cache), _seqs(**seqs)
    with pytest.raises(fz.FurnaceError, match=words) as e:
        c.append(s, a["x"], FAKE, a["ld"], dtype=a["dtype"])
    assert e.value.code == fz.FZ_EINVAL
    if "x" not in args:  # read takes a null k
        with pytest.raises(fz.FurnaceError, match=words):
            c.read(s, a["x"], FAKE, a["ld"], dtype=a["dtype"])
    with pytest.raises(fz.FurnaceError, match=words):
        c.attend(s, a["x"], FAKE + (1 << 16), a["ld"] * 4 if a["ld"] == 128 else a["ld"], 512, FAKE, 1 << 30,
                 dtype=a["dtype"])


def test_attend_refusals():
    c, s = _cache(), _seqs()
    n = c.attend_work(s)
    for args, words in ((dict(work=None), "work"), (dict(work=FAKE + 8), "work"), (dict(work_bytes=n - 1), "work"),
                        (dict(out=FAKE), "overlap"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
                        (dict(ldo=511), "16-byte"), (dict(ldq=508), "row stride"), (dict(out=None), "null")):
        a = dict(q=FAKE, out=FAKE + (1 << 16), ldq=512, ldo=512, work=FAKE, work_bytes=n)
        a.update(args)
        with pytest.raises(fz.FurnaceError, match=words) as e:
            c.attend(s, **a)
        assert e.value.code == fz.FZ_EINVAL
    L = fz.load_library()
    assert L.fz_kvq8_attend_work(c._p, s._p, None) == fz.FZ_EINVAL
    assert L.fz_kvq8_append_dev(None, s._p, 0, FAKE, FAKE, 128, None) == fz.FZ_EINVAL
    assert L.fz_kvq8_append_dev(c._p, None, 0, FAKE, FAKE, 128, None) == fz.FZ_EINVAL


def test_calls_without_rows_are_no_work():
    """No sequences or no rows: nothing is queued, so this runs without a GPU."""
    c = _cache()
    for s in (_seqs(n_seqs=0, pages=None, lens=None, starts=None, n_rows=0), _seqs(n_rows=0)):
        c.append(s, None, None, 128)
        c.read(s, None, None, 128)
        c.attend(s, None, None, 512, 512, None, 0)


# ---------------------------------------------------------------------------
# On the GPU
# ---------------------------------------------------------------------------
class Dev:
    """A cache on the device next to its restatement."""

    def __init__(self, n_pages, heads, kv, hd, n_rope=0, seed=0, first_page=0):
        import torch

        self.t, self.kv, self.hd, self.heads = torch, kv, hd, heads
        self.rng = np.random.default_rng(seed)
        self.plain = Plain(n_pages, kv, hd, rope_table(n_rope, hd) if n_rope else None)
        self.n_pages = n_pages
        # what no call has written is garbage: any byte, scales that are no numbers
        self.codes = torch.randint(0, 256, (first_page + n_pages, kv, 2, PAGE * hd), dtype=torch.uint8, device="cuda")
        self.scales = torch.full((first_page + n_pages, kv, 2, 4), float("nan"), device="cuda")
        self.first = first_page
        self.rope = torch.from_numpy(self.plain.rope).cuda() if n_rope else None
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.c = fz.KvQ8(self.codes.data_ptr(), self.scales.data_ptr(), self.status.data_ptr(), first_page + n_pages,
                         heads, kv, hd, rope=self.rope.data_ptr() if n_rope else None, n_rope=n_rope)
        self.order = self.rng.permutation(n_pages)
        self.used = 0

    def table(self, lens, spare=0):
        """A page table with fresh pages; entries past a sequence's end are out of range."""
        need = [(n + PAGE - 1) // PAGE for n in lens]
        t = np.full((len(lens), max(max(need), 1) + spare), -7, np.int32)
        for i, n in enumerate(need):
            t[i, :n] = self.order[self.used:self.used + n]
            self.used += n
        assert self.used <= self.n_pages
        return t

    def stream(self):
        return self.t.cuda.current_stream().cuda_stream

    def seqs(self, table, lens, news, n_rows=None, uniform=False):
        ints = lambda x: self.t.tensor(np.asarray(x, np.int32)).cuda()
        starts = np.concatenate([[0], np.cumsum(news)])
        hold = (ints(np.where(table >= 0, table + self.first, table)), ints(lens), ints(starts))
        s = fz.KvQ8Seqs(hold[0].data_ptr(), hold[1].data_ptr(), len(lens), table.shape[1],
                        n_rows if n_rows is not None else int(starts[-1]),
                        starts=None if uniform else hold[2].data_ptr(), max_new=max(1, int(max(news))))
        s.hold = hold
        return s

    def rows(self, n, heads, dtype, ld=None, spread=1.0):
        """n rows of heads (numpy f32 values that dtype holds, device buffer with row stride ld)."""
        x = (self.rng.standard_normal((n, heads, self.hd)) * spread).astype(np.float32)
        if dtype == fz.F16:
            x = x.astype(np.float16).astype(np.float32)
        ld = ld or heads * self.hd
        td = self.t.float16 if dtype == fz.F16 else self.t.float32
        d = self.t.full((n, ld), 7.0, dtype=td, device="cuda")
        d[:, :heads * self.hd] = self.t.from_numpy(x.reshape(n, -1)).cuda().to(td)
        return x, d

    def append(self, table, lens, news, dtype=fz.F32, k=None, v=None, uniform=False):
        n = int(sum(news))
        k = k or self.rows(n, self.kv, dtype)
        v = v or self.rows(n, self.kv, dtype)
        s = self.seqs(table, lens, news, uniform=uniform)
        self.c.append(s, k[1].data_ptr(), v[1].data_ptr(), k[1].shape[1], dtype=dtype, stream=self.stream())
        r = 0
        for i, (length, new) in enumerate(zip(lens, news)):
            if new:
                self.plain.append(table[i], length, k[0][r:r + new], v[0][r:r + new])
            r += new
        return s

    def attend(self, table, lens, news, dtype=fz.F32, q=None, uniform=False, **kw):
        n = int(sum(news))
        q = q or self.rows(n, self.heads, dtype)
        s = self.seqs(table, lens, news, uniform=uniform)
        work = self.t.full((self.c.attend_work(s),), 0xFF, dtype=self.t.uint8, device="cuda")  # NaNs
        out = self.t.full((n, self.heads, self.hd), 99.0, dtype=q[1].dtype, device="cuda")
        self.c.attend(s, q[1].data_ptr(), out.data_ptr(), q[1].shape[1], self.heads * self.hd, work.data_ptr(),
                      work.numel(), dtype=dtype, stream=self.stream(), **kw)
        self.t.cuda.synchronize()
        return q[0], out.float().cpu().numpy()

    def check_attend(self, table, lens, news, dtype=fz.F32, **kw):
        q, got = self.attend(table, lens, news, dtype, **kw)
        kw = {k: v for k, v in kw.items() if k in ("window", "sinks", "scale")}
        r = 0
        for i, (length, new) in enumerate(zip(lens, news)):
            want, tol = self.plain.attend(table[i], length, q[r:r + new], **kw)
            if dtype == fz.F16:
                tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25  # half a step, normal and subnormal
            err = np.abs(got[r:r + new] - want)
            assert (err <= tol).all(), (i, length, new, float((err / tol).max()), float(err.max()))
            r += new
        self.c.status(self.stream())

    def check_cache(self, written):
        """Codes and scales of the blocks holding `written` (table row, length) equal the restatement's."""
        codes = self.codes.cpu().numpy()[self.first:].reshape(self.n_pages, self.kv, 2, PAGE // BLOCK, BLOCK * self.hd)
        scales = self.scales.cpu().numpy()[self.first:]
        ki, vi = block_index(self.hd)
        for row, length in written:
            for b in range((length + BLOCK - 1) // BLOCK):
                page, sub, n = row[b * BLOCK // PAGE], b % (PAGE // BLOCK), min(BLOCK, length - b * BLOCK)
                assert np.array_equal(scales[page, :, :, sub], self.plain.scales[page, :, :, sub]), (b, page)
                for w, at in ((0, ki), (1, vi)):
                    got = codes[page, :, w, sub][:, at[:n]].astype(np.int32) - 128
                    assert np.array_equal(got, self.plain.codes[page, :, w, sub, :n]), (b, page, w)


@pytest.fixture(scope="module")
def gpu():
    from tests.conftest import gpu_available

    if not gpu_available():
        pytest.fail("GPU tests need a CUDA device")
    import torch

    fz.load_library()
    return torch


LENS = [1, 2, 15, 16, 17, 63, 64, 65, 130, 200]


@pytest.mark.gpu
@pytest.mark.parametrize("hd, kv, dtype, n_rope", [(64, 1, fz.F32, 256), (128, 3, fz.F32, 256), (128, 2, fz.F16, 256),
                                                   (64, 2, fz.F16, 0), (128, 1, fz.F32, 0)])
def test_append_whole_sequences(gpu, hd, kv, dtype, n_rope):
    d = Dev(40, kv, kv, hd, n_rope)
    t = d.table(LENS)
    d.append(t, LENS, LENS, dtype)
    gpu.cuda.synchronize()
    d.check_cache(zip(t, LENS))
    d.c.status(d.stream())


@pytest.mark.gpu
@pytest.mark.parametrize("hd, dtype", [(64, fz.F32), (128, fz.F16)])
def test_append_in_pieces_rescales_older_codes(gpu, hd, dtype):
    """Pieces of 1..20 positions, values growing from call to call, so that
    blocks are entered in the middle and their scales grow, and shrinking, so
    that they stay; one sequence gets nothing in some calls."""
    d = Dev(16, 2, 2, hd, 256)
    final = [70, 33, 64]
    t = d.table(final)
    at = [0, 0, 0]
    rng = np.random.default_rng(5)
    step = 0
    while at != final:
        news = [min(f - a, int(n)) for f, a, n in zip(final, at, rng.integers(0, 20, 3))]
        if step % 3 == 0:
            news = [min(f - a, 1) for f, a in zip(final, at)]
        step += 1
        if not sum(news):
            continue
        at = [a + n for a, n in zip(at, news)]
        n = sum(news)
        spread = [0.1, 3.0, 1.0, 10.0][step % 4]
        d.append(t, at, news, dtype, k=d.rows(n, 2, dtype, spread=spread), v=d.rows(n, 2, dtype, spread=spread))
    gpu.cuda.synchronize()
    d.check_cache(zip(t, final))


@pytest.mark.gpu
def test_append_zeros_rewinds_and_strides(gpu):
    """All-zero values, a rewound sequence written again, and k and v as
    columns of one wide row."""
    d = Dev(8, 4, 2, 128, 128)
    t = d.table([100])
    zero = (np.zeros((50, 2, 128), np.float32), gpu.zeros(50, 256, device="cuda"))
    d.append(t, [50], [50], k=zero, v=zero)
    d.check_attend(t, [50], [3])
    qkv = gpu.full((30, 4 * 128 + 2 * 2 * 128), 5.0, device="cuda")
    x = d.rng.standard_normal((30, 2, 2, 128)).astype(np.float32)
    qkv[:, 512:] = gpu.from_numpy(x.reshape(30, -1)).cuda()
    s = d.seqs(t, [55], [30])  # positions 25 .. 54 again
    d.c.append(s, qkv.data_ptr() + 512 * 4, qkv.data_ptr() + 768 * 4, 1024, stream=d.stream())
    d.plain.append(t[0], 55, x[:, 0], x[:, 1])
    gpu.cuda.synchronize()
    d.check_cache([(t[0], 55)])
    d.check_attend(t, [55], [7])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [fz.F32, fz.F16])
def test_read_back(gpu, dtype):
    d = Dev(12, 2, 2, 64, 256)
    lens = [130, 0, 17]
    t = d.table(lens)
    d.append(t, lens, lens)
    news = [100, 0, 17]
    s = d.seqs(t, lens, news, n_rows=119)
    td = gpu.float16 if dtype == fz.F16 else gpu.float32
    k, v = (gpu.full((119, 136), 3.0, dtype=td, device="cuda") for _ in range(2))
    d.c.read(s, k.data_ptr(), v.data_ptr(), 136, dtype=dtype, stream=d.stream())
    only = gpu.full_like(k, 3.0)
    d.c.read(s, only.data_ptr(), None, 136, dtype=dtype, stream=d.stream())
    gpu.cuda.synchronize()
    assert gpu.equal(only, k)
    for which, got in enumerate((k, v)):
        want = np.concatenate([d.plain.rows(t[0], 30, 130, np.float32)[which].transpose(1, 0, 2),
                               d.plain.rows(t[2], 0, 17, np.float32)[which].transpose(1, 0, 2)]).reshape(117, 128)
        want = gpu.from_numpy(want).to(td)
        assert gpu.equal(got[:117, :128].cpu(), want)
        assert (got[117:] == 3.0).all() and (got[:, 128:] == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hd, kv, group, dtype", [(64, 2, 1, fz.F32), (64, 1, 7, fz.F16), (128, 2, 4, fz.F32),
                                                  (128, 1, 8, fz.F32), (128, 4, 7, fz.F16), (128, 1, 12, fz.F32),
                                                  (64, 1, 40, fz.F32)])
@pytest.mark.parametrize("new", [1, 3])
def test_attend_lengths(gpu, hd, kv, group, dtype, new):
    d = Dev(60, kv * group, kv, hd, 600)
    lens = [n for n in LENS + [512, 577] if n >= new]
    t = d.table(lens)
    d.append(t, lens, lens)
    d.check_attend(t, lens, [new] * len(lens), dtype, uniform=new == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("hd, kv, group, dtype", [(128, 2, 7, fz.F32), (128, 1, 5, fz.F16), (64, 2, 8, fz.F32),
                                                  (64, 1, 1, fz.F16)])
def test_attend_prompts(gpu, hd, kv, group, dtype):
    """Whole prompts, prompts behind a prefix, sequences without new rows or positions."""
    d = Dev(60, kv * group, kv, hd, 1200)
    lens, news = [300, 200, 1000, 0, 65, 17, 128], [300, 71, 130, 0, 0, 17, 128]
    t = d.table(lens)
    d.append(t, lens, lens)
    d.check_attend(t, lens, news, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (7, 0), (16, 3), (64, 4), (65, 70), (200, 16), (5000, 4),
                                           (2 ** 32 - 1, 2 ** 32 - 1), (30, 2 ** 32 - 1)])
@pytest.mark.parametrize("new", [1, 4, 90])
def test_attend_window(gpu, window, sinks, new):
    d = Dev(40, 14, 2, 64, 1000)
    lens = [n for n in [1, 40, 64, 100, 333, 900] if n >= new]
    t = d.table(lens)
    d.append(t, lens, lens)
    d.check_attend(t, lens, [new] * len(lens), window=window, sinks=sinks)


@pytest.mark.gpu
def test_attend_scales_far_apart(gpu):
    """Blocks whose values differ by many powers of two, huge scores, a given
    softmax scale, no rotation."""
    d = Dev(20, 8, 2, 128)
    lens = [16 * 12]
    t = d.table(lens)
    for b in range(12):
        k = d.rows(16, 2, fz.F32, spread=[1.0, 8.0, 0.01][b % 3])
        v = d.rows(16, 2, fz.F32, spread=10.0 ** (b - 6))
        d.append(t, [16 * (b + 1)], [16], k=k, v=v)
    d.check_attend(t, lens, [1])
    d.check_attend(t, lens, [5], scale=1.5)
    d.check_attend(t, lens, [100], scale=-0.02)
    d.check_attend(t, lens, [2], q=d.rows(2, 8, fz.F32, spread=1e-20))
    d.check_attend(t, lens, [2], q=d.rows(2, 8, fz.F32, spread=2e4), scale=1e-5)


@pytest.mark.gpu
def test_attend_tiny_and_huge_values(gpu):
    """Values near the ends of f32's range keep their relative precision."""
    for spread in (1e-25, 1e30):
        d = Dev(4, 4, 2, 64, 100)
        t = d.table([90])
        d.append(t, [90], [90], v=d.rows(90, 2, fz.F32, spread=spread))
        d.check_attend(t, [90], [1])
        d.check_attend(t, [90], [33])


@pytest.mark.gpu
def test_rows_of_no_sequence_stay(gpu):
    d = Dev(10, 8, 2, 128, 200)
    lens = [100, 64]
    t = d.table(lens)
    d.append(t, lens, lens)
    s = d.seqs(t, lens, [1, 1], n_rows=6)
    q, out = d.rows(6, 8, fz.F32), gpu.full((6, 1024), 99.0, device="cuda")
    work = gpu.empty(d.c.attend_work(s), dtype=gpu.uint8, device="cuda")
    d.c.attend(s, q[1].data_ptr(), out.data_ptr(), 1024, 1024, work.data_ptr(), work.numel(), stream=d.stream())
    gpu.cuda.synchronize()
    assert (out[2:] == 99.0).all() and not (out[:2] == 99.0).any()
    # a row whose sequence holds no positions: starts may say so only with 0 rows
    d.c.status(d.stream())


@pytest.mark.gpu
def test_offsets_beyond_32_bits(gpu):
    """Pages whose bytes lie past 4 GB of the pool."""
    d = Dev(12, 16, 8, 128, 300, first_page=(1 << 32) // fz.KvQ8.page_bytes(8, 128))
    lens = [250, 70]
    t = d.table(lens)
    d.append(t, lens, lens)
    gpu.cuda.synchronize()
    d.check_cache(zip(t, lens))
    d.check_attend(t, lens, [1, 1], uniform=True)
    d.check_attend(t, lens, [60, 70])
    del d
    gpu.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["len", "len<0", "rows", "row0", "page", "page<0", "rope", "new>len"])
def test_bad_numbers_are_reported_and_touch_nothing_else(gpu, what):
    """The second of three sequences has a number out of range: the others'
    results are as without it, the call's status names it, and the next call
    is clean."""
    d = Dev(12, 4, 2, 64, 150)
    lens, news = [100, 90, 40], [2, 3, 1]
    t = d.table(lens, spare=1)
    d.append(t, lens, lens)
    d.c.status(d.stream())
    bad_t, bad_lens, bad_news, rows = t.copy(), list(lens), list(news), 6
    words = "lengths or rows"
    if what == "len":
        bad_lens[1] = 3 * PAGE + 1
    elif what == "len<0":
        bad_lens[1] = -1
    elif what == "page":
        bad_t[1, 1], words = d.n_pages, "page number"
    elif what == "page<0":
        bad_t[1, 1], words = -2 ** 31, "page number"
    elif what == "rope":
        bad_lens[1], words = 151, "rotation table"
        bad_t[1] = d.order[d.used:d.used + 3]
    elif what == "new>len":
        bad_lens[1] = 2
    s = d.seqs(bad_t, bad_lens, bad_news, n_rows=rows)
    if what == "rows":
        s.hold[2].copy_(gpu.tensor([0, 2, 2 + 900, 6]))
    elif what == "row0":
        s.hold[2].copy_(gpu.tensor([0, 2, -1, 1]))
    if what in ("rows", "row0"):  # the third sequence's rows are then given by the same table: leave it out too
        check = [0]
    else:
        check = [0, 2]
    before = (d.codes.clone(), d.scales.clone())
    q, out = d.rows(6, 4, fz.F32), gpu.full((6, 256), 99.0, device="cuda")
    work = gpu.empty(d.c.attend_work(s), dtype=gpu.uint8, device="cuda")
    d.c.attend(s, q[1].data_ptr(), out.data_ptr(), 256, 256, work.data_ptr(), work.numel(), stream=d.stream())
    with pytest.raises(fz.FurnaceError, match=words) as e:
        d.c.status(d.stream())
    assert e.value.code == fz.FZ_EINVAL
    d.c.status(d.stream())  # reported once
    assert gpu.equal(d.codes, before[0]) and gpu.equal(d.scales.view(gpu.int32), before[1].view(gpu.int32))
    got = out.view(6, 4, 64).cpu().numpy()
    for i in check:
        r = sum(news[:i])
        want, tol = d.plain.attend(t[i], lens[i], q[0][r:r + news[i]])
        assert (np.abs(got[r:r + news[i]] - want) <= tol).all()
    k = d.rows(6, 2, fz.F32)
    d.c.append(s, k[1].data_ptr(), k[1].data_ptr(), 128, stream=d.stream())
    with pytest.raises(fz.FurnaceError, match=words):
        d.c.status(d.stream())
    out16 = gpu.full((6, 128), 5.0, device="cuda")
    d.c.read(s, out16.data_ptr(), None, 128, stream=d.stream())
    if what != "rope":
        with pytest.raises(fz.FurnaceError, match=words):
            d.c.status(d.stream())
    # the untouched sequences hold what they held, with the new rows appended
    for i in check:
        r = sum(news[:i])
        d.plain.append(t[i], lens[i], k[0][r:r + news[i]], k[0][r:r + news[i]])
    gpu.cuda.synchronize()
    d.check_cache([(t[i], lens[i]) for i in check])


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite_are_reported(gpu, value):
    d = Dev(4, 2, 1, 64, 100)
    t = d.table([40])
    d.append(t, [20], [20])
    k, v = d.rows(20, 1, fz.F32), d.rows(20, 1, fz.F32)
    v[1][15, 3] = value  # position 35: block 2
    s = d.seqs(t, [40], [20])
    d.c.append(s, k[1].data_ptr(), v[1].data_ptr(), 64, stream=d.stream())
    with pytest.raises(fz.FurnaceError, match="not finite"):
        d.c.status(d.stream())
    scales = d.scales[t[0, 0]].cpu()
    assert scales[0, 1, 2].isnan() and scales[0, 1, :2].isfinite().all() and scales[0, 0, :3].isfinite().all()
    # positions that see the block get no number, those that do not are as before
    s = d.seqs(t, [40], [40])
    q, out = d.rows(40, 2, fz.F32), gpu.zeros(40, 128, device="cuda")
    work = gpu.empty(d.c.attend_work(s), dtype=gpu.uint8, device="cuda")
    d.c.attend(s, q[1].data_ptr(), out.data_ptr(), 128, 128, work.data_ptr(), work.numel(), stream=d.stream())
    gpu.cuda.synchronize()
    assert out[:32].isfinite().all() and out[32:].isnan().all()


@pytest.mark.gpu
def test_decode_loop_captured_and_replayed(gpu):
    """append + attend of three sequences in one graph on a side stream; each
    replay takes the next rows and lengths from the same buffers."""
    d = Dev(20, 14, 2, 128, 300)
    lens = [60, 15, 200]
    t = d.table([n + 10 for n in lens])
    d.append(t, lens, lens)
    s = d.seqs(t, lens, [1, 1, 1], uniform=True)
    kbuf, vbuf, qbuf = (gpu.zeros(3, n * 128, device="cuda") for n in (2, 2, 14))
    out = gpu.zeros(3, 14 * 128, device="cuda")
    work = gpu.empty(d.c.attend_work(s), dtype=gpu.uint8, device="cuda")
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())

    def step(stream):
        s.hold[1].add_(1)
        d.c.append(s, kbuf.data_ptr(), vbuf.data_ptr(), 256, stream=stream)
        d.c.attend(s, qbuf.data_ptr(), out.data_ptr(), 1792, 1792, work.data_ptr(), work.numel(), stream=stream)

    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph, stream=side):
        step(gpu.cuda.current_stream().cuda_stream)
    gpu.cuda.synchronize()
    for i in range(6):
        k, v, q = (d.rng.standard_normal((3, n, 128)).astype(np.float32) for n in (2, 2, 14))
        for buf, x in ((kbuf, k), (vbuf, v), (qbuf, q)):
            buf.copy_(gpu.from_numpy(x.reshape(3, -1)))
        graph.replay()
        gpu.cuda.synchronize()
        lens = [n + 1 for n in lens]
        for j, n in enumerate(lens):
            d.plain.append(t[j], n, k[j:j + 1], v[j:j + 1])
            want, tol = d.plain.attend(t[j], n, q[j:j + 1])
            assert (np.abs(out[j].view(1, 14, 128).cpu().numpy() - want) <= tol).all(), (i, j)
    d.check_cache(zip(t, lens))
    d.c.status(side.cuda_stream)


@pytest.mark.gpu
def test_two_streams_and_repeated_calls_give_the_same_bits(gpu):
    d = Dev(300, 28, 4, 128, 4000)
    lens = [3900, 700, 1500, 33]
    t = d.table(lens)
    d.append(t, lens, lens)
    s = d.seqs(t, lens, [1] * 4, uniform=True)
    p = d.seqs(t, lens, [200, 100, 300, 33])
    q1, q2 = d.rows(4, 28, fz.F32)[1], d.rows(633, 28, fz.F32)[1]
    outs = []
    gpu.cuda.synchronize()
    for i in range(4):
        st = gpu.cuda.Stream()
        for seqs, q in ((s, q1), (p, q2)):
            work = gpu.full((d.c.attend_work(seqs),), 255, dtype=gpu.uint8, device="cuda")
            out = gpu.zeros_like(q)
            gpu.cuda.synchronize() if i == 0 else st.wait_stream(gpu.cuda.current_stream())
            d.c.attend(seqs, q.data_ptr(), out.data_ptr(), 28 * 128, 28 * 128, work.data_ptr(), work.numel(),
                       stream=st.cuda_stream)
            outs.append((out, work))
    gpu.cuda.synchronize()
    for i in range(2, 8):
        assert gpu.equal(outs[i][0], outs[i % 2][0])
