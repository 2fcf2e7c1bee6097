"""FZ_KV_Q8 caches under tensor parallelism on 2 GPUs against the oracle with
the same cache: a prompt, a second one from the middle of a block, greedy steps,
with and without a window.  Needs two visible GPUs; skipped otherwise.  Bars as
for one GPU (tests/test_kvq8_model.py)."""

import os

import numpy as np
import pytest

import furnace_b200 as fz
from furnace_b200 import synth
from tests.test_kvq8_model import LOGIT_ABS, _oracle_prompt
from tests.test_tp_gpu import _ngpus, _spawn

pytestmark = pytest.mark.gpu
WORLD, PROMPTS, STEPS, CTX = 2, ((100, 41), (45, 42)), 16, 200


@pytest.fixture(scope="module", autouse=True)
def _two_gpus():
    if _ngpus() < 2:
        pytest.skip("tensor parallelism needs two GPUs")


def _rank(rank, world, port, path, window, sinks, q):
    import torch.distributed as dist

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), NCCL_NVLS_ENABLE="0")
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        ids = [fz.tp_unique_id() if rank == 0 else None]
        dist.broadcast_object_list(ids, src=0)
        m = fz.Model.load_tp(fz.GgufFile.open(path), rank, world, ids[0], rank)
        kv = fz.KvCache(m, CTX, fz.FZ_KV_Q8)
        if window:
            kv.set_window(window, sinks)
        prompts = [m.forward(synth.prompt_ids(m.config.vocab, n, seed=s), kv) for n, s in PROMPTS]
        n = sum(n for n, _ in PROMPTS)
        rows = [kv.read(0, w, n) for w in (0, 1)]
        steps = m.decode_greedy(prompts[-1][1], STEPS, kv, keep_logits=True)
        q.put((rank, (prompts, rows, steps), None))
        kv.close()
        m.close()
        dist.barrier()
    except Exception as e:  # reported to the parent, which fails the test
        q.put((rank, repr(e), None))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("over", [{}, {"hidden": 768, "n_heads": 12}], ids=["tiny", "tiny-768"])
@pytest.mark.parametrize("window, sinks", [(0, 0), (24, 4)])
def test_tp2_matches_the_oracle(orc, tmp_path, over, window, sinks):
    """With 12 heads of 64 each rank's o_proj input (384 columns) widens to whole
    256-element blocks in odd layers, so the attention's output sits at an offset
    inside zero padding."""
    path, world = synth.write(synth.spec("tiny", **over), str(tmp_path / "m.gguf")), WORLD
    res = _spawn(_rank, world, path, window, sinks)
    ref = orc.Model(path)
    kr = ref.kv_new(CTX, kv_dtype=2)
    if window:
        kr.set_window(window, sinks)
    for i, (n, seed) in enumerate(PROMPTS):
        want = _oracle_prompt(ref, synth.prompt_ids(ref.vocab, n, seed=seed), kr)
        for r in range(world):
            assert np.abs(res[r][0][i][0] - want).max() <= LOGIT_ABS, (r, i)
    n, per = sum(n for n, _ in PROMPTS), ref.n_kv_heads // world * ref.head_dim
    for r in range(world):
        for w in (0, 1):
            a, b = res[r][1][w], kr.read(0, w, n)[:, r * per:(r + 1) * per]
            top = np.abs(b).max()
            assert np.abs(a - b).max() <= 2.02 * top / 127 + 1e-4 * top
            assert np.mean(np.abs(a - b) <= 1e-4 * top) > 0.97
    assert res[0][2][0].tolist() == res[world - 1][2][0].tolist()  # every rank takes the same tokens
    ids, lg = res[0][2]
    for step in range(STEPS - 1):  # the oracle takes the device's tokens: near ties may go either way
        assert want.max() - want[ids[step]] <= 2 * LOGIT_ABS, step
        want = ref.forward_cached([int(ids[step])], kr)
        assert np.abs(lg[step] - want).max() <= LOGIT_ABS, step
