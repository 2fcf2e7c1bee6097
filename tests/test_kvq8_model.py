"""FZ_KV_Q8 caches: the model's prefill and decode on 8-bit codes, with and
without a sliding window, against the oracle with the same cache.

A cached element may land one code apart: device and oracle feed the
quantizer values that differ by GEMV rounding.  The bar for those is 1e-4 of
the largest, 0.013 of a code, so that at most 2.6 % of the elements can differ;
the measured rounding is 50 times smaller.  One code is 1/127 of a block's
largest magnitude, about 0.03 of a standard deviation; with 0.05 % of a head's
elements off by that and weights of 1 / 40 a position, the attention's output
moves by about 5e-4 of itself in a layer, the logits (of order 1) of three
layers by 1.5e-3: their bar here is 5e-3.
"""

import numpy as np
import pytest

import furnace_b200 as fz
from furnace_b200 import synth

LOGIT_ABS = 5e-3


def _oracle_prompt(ref, ids, cache):
    """The device appends a prompt's last token by itself (it produces the
    logits), and one of up to 8 tokens one by one; a block's scale goes by
    what one call appends."""
    if len(ids) > 8:
        ref.forward_cached(ids[:-1], cache)
        return ref.forward_cached(ids[-1:], cache)
    for t in ids:
        lg = ref.forward_cached([t], cache)
    return lg


def _check_rows(kd, kr, n_layers, n):
    for layer in range(n_layers):
        for which in (0, 1):
            a, b = kd.read(layer, which, n), kr.read(layer, which, n)
            top = max(1e-30, float(np.abs(b).max()))
            off = np.abs(a - b)
            # a row appended into a block that was rescaled later was rounded twice
            assert off.max() <= 2.02 * top / 127 + 1e-4 * top, (layer, which, off.max() / top)
            # 2 x 0.013 of the elements at most differ in the first layer.  Later layers' inputs carry the codes that
            # differ before them: 5e-4 of the attention's output (see above) is 5e-4 of a standard deviation, more than
            # the 1e-4 of the largest element (3.5e-4) that counts as equal here, so the share says nothing there.
            if layer == 0:
                assert np.mean(off <= 1e-4 * top) > 0.97, (layer, which)


def test_oracle_q8_cache_follows_the_f32_cache(orc, tmp_path):
    """The oracle's own 8-bit cache: rows within half a code (twice rounded:
    one) of the f32 cache's in the first layer, whose inputs are the same; a
    window that covers everything changes nothing, a small one does."""
    ref = orc.Model(synth.write(synth.spec("tiny"), str(tmp_path / "m.gguf")))
    ids = synth.prompt_ids(ref.vocab, 40, seed=3)
    k32, k8, kw, ks = (ref.kv_new(64, kv_dtype=t) for t in (0, 2, 2, 2))
    kw.set_window(64, 0)
    ks.set_window(8, 2)
    a, b, c, d = (_oracle_prompt(ref, ids, k) for k in (k32, k8, kw, ks))
    for which in (0, 1):
        x, y = k32.read(0, which, 40), k8.read(0, which, 40)
        assert np.abs(x - y).max() <= 1.01 * np.abs(x).max() / 127
        assert not np.array_equal(x, y)
    assert np.array_equal(b, c) and not np.allclose(b, d, atol=1e-3)
    assert np.abs(a - b).max() < 0.5  # the 8-bit cache is an approximation, not another model


@pytest.fixture(scope="module")
def gpu():
    from tests.conftest import gpu_available

    if not gpu_available():
        pytest.fail("GPU tests need a CUDA device")
    fz.load_library()


def _models(orc, path):
    return fz.Model.load(fz.GgufFile.open(path)), orc.Model(path)


SHAPES = [{}, {"hidden": 1792, "n_heads": 14, "n_kv_heads": 2}]


@pytest.mark.gpu
@pytest.mark.parametrize("over", SHAPES, ids=["hd64-g4", "hd128-g7"])
@pytest.mark.parametrize("window, sinks", [(0, 0), (24, 4)])
def test_prompts_and_decode_match_the_oracle(gpu, orc, tmp_path, over, window, sinks):
    """A prompt, a second one from the middle of a block, then 24 greedy steps."""
    dev, ref = _models(orc, synth.write(synth.spec("tiny", **over), str(tmp_path / "m.gguf")))
    kd, kr = fz.KvCache(dev, 300, fz.FZ_KV_Q8), ref.kv_new(300, kv_dtype=2)
    if window:
        kd.set_window(window, sinks)
        kr.set_window(window, sinks)
    n = 0
    for count, seed in ((150, 31), (75, 32), (3, 33)):
        ids = synth.prompt_ids(ref.vocab, count, seed=seed)
        got, am = dev.forward(ids, kd)
        want = _oracle_prompt(ref, ids, kr)
        assert np.abs(got - want).max() <= LOGIT_ABS, (count, np.abs(got - want).max())
        n += count
    _check_rows(kd, kr, ref.n_layers, n)
    ids, lg = dev.decode_greedy(am, 24, kd, keep_logits=True)
    tok = int(np.argmax(want))
    for step in range(24):
        top = np.sort(want)[-2:]
        if top[1] - top[0] <= 2 * LOGIT_ABS:
            break  # the two sides may well pick another token from here on
        assert ids[step] == tok, step
        if step == 23:
            break
        want = ref.forward_cached([tok], kr)
        assert np.abs(lg[step] - want).max() <= LOGIT_ABS, step
        tok = int(np.argmax(want))
    assert step > 2
    assert kd.len == n + 23


@pytest.mark.gpu
def test_one_kv_head_and_long_context(gpu, orc, tmp_path):
    """Every run of the split attention has work: one KV head for 8 query
    heads, 700 positions."""
    dev, ref = _models(orc, synth.write(synth.spec("tiny", n_kv_heads=1), str(tmp_path / "m.gguf")))
    kd, kr = fz.KvCache(dev, 800, fz.FZ_KV_Q8), ref.kv_new(800, kv_dtype=2)
    ids = synth.prompt_ids(ref.vocab, 700, seed=5)
    got, _ = dev.forward(ids, kd)
    assert np.abs(got - _oracle_prompt(ref, ids, kr)).max() <= LOGIT_ABS
    for t in ids[:20]:
        got = dev.forward_cached([t], kd)
        assert np.abs(got - ref.forward_cached([t], kr)).max() <= LOGIT_ABS
    _check_rows(kd, kr, ref.n_layers, 720)


@pytest.mark.gpu
def test_rewind_reset_bytes_and_window_changes(gpu, orc, tmp_path):
    path = synth.write(synth.spec("tiny"), str(tmp_path / "m.gguf"))
    dev, ref = _models(orc, path)
    c = dev.config
    kd, kr = fz.KvCache(dev, 100, fz.FZ_KV_Q8), ref.kv_new(100, kv_dtype=2)
    assert kd.bytes() == c.n_layers * 2 * 2 * c.n_kv_heads * (64 * c.head_dim + 4 * 4)
    assert not kd.read(0, False, 100).any()
    ids = synth.prompt_ids(ref.vocab, 60, seed=9)
    a, _ = dev.forward(ids, kd)
    kd.reset()
    b, _ = dev.forward(ids, kd)
    assert np.array_equal(a, b)
    _oracle_prompt(ref, ids, kr)
    kd.len = kr.len = 37  # into the middle of a block, whose scale stays at least what it was
    more = synth.prompt_ids(ref.vocab, 20, seed=10)
    got, _ = dev.forward(more, kd)
    assert np.abs(got - _oracle_prompt(ref, more, kr)).max() <= LOGIT_ABS
    _check_rows(kd, kr, ref.n_layers, 57)
    # the captured step follows a window that changes between steps
    for window, sinks in ((10, 2), (0, 0), (1, 0), (1000, 7)):
        kd.set_window(window, sinks)
        kr.set_window(window, sinks)
        got = dev.forward_cached([5], kd)
        assert np.abs(got - ref.forward_cached([5], kr)).max() <= LOGIT_ABS, (window, sinks)
    with pytest.raises(fz.FurnaceError, match="sinks without a window") as e:
        kd.set_window(0, 3)
    assert e.value.code == fz.FZ_EINVAL
    with pytest.raises(fz.FurnaceError, match="8-bit cache"):
        fz.KvCache(dev, 16).set_window(4)
    with pytest.raises(fz.FurnaceError, match="kv dtype 3"):
        fz.KvCache(dev, 16, 3)
    with pytest.raises(fz.FurnaceError, match="context overflow"):
        dev.forward(synth.prompt_ids(ref.vocab, 60, seed=1), kd)
    prof = dev.step_profile(3, 2, kd)
    assert prof["attention"][2] == 2 * c.n_layers and prof["attention"][0] > 0
    dev.close()
    with pytest.raises(fz.FurnaceError, match="freed"):
        kd.set_window(3, 0)
    kd.close()


@pytest.mark.gpu
def test_generate_with_an_8_bit_cache(gpu, orc, tmp_path):
    """generate and generate_sampled take the cache type and the window; an
    8-bit cache of a window over everything gives the same ids as none."""
    dev, ref = _models(orc, synth.write(synth.spec("tiny"), str(tmp_path / "m.gguf")))
    ids = synth.prompt_ids(ref.vocab, 30, seed=2)
    a, _ = fz.generate(dev, ids, 12, max_ctx=64, kv_dtype=fz.FZ_KV_Q8)
    b, _ = fz.generate(dev, ids, 12, max_ctx=64, kv_dtype=fz.FZ_KV_Q8, window=64, sinks=1)
    assert a.tolist() == b.tolist()
    s = [fz.generate_sampled(dev, ids, 12, fz.Sampler(0.8, 20, 0.9, 1.1, 7), max_ctx=64, kv_dtype=fz.FZ_KV_Q8,
                             window=w, sinks=0) for w in (0, 64)]
    assert s[0].tolist() == s[1].tolist() and len(s[0]) == 12
