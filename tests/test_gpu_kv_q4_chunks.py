"""Chunks over a 4-bit cache whose values are beyond what f16 holds (65504): the tier keeps values up to 8 * 65504, and one-token steps and the
read-back have them. Held to the tolerance of test_gpu_long_context.py, which this takes its plain model from."""
import numpy as np
import pytest

import effect_torch_b200 as et
import oracle as orc
from tests import helpers
from tests.test_gpu_long_context import PAGE, SMALL_Q, WIDE_Q, dense, make

pytestmark = pytest.mark.gpu
PAIRS = dict(layout=et.INTERLEAVED_PAIRS)  # a rotated pair lies in one block


def weights(cfg, keys, values):
    """`keys`: the first block of the first KV head's keys is large, and the queries have zeros there. `values`: the second block of the last
    KV head's values is large, and what comes of it is made small again by the output projection."""
    w = helpers.make_weights(cfg, seed=3)
    layer, D, G = w["layers"][0], cfg["head_dim"], cfg["q_heads"] // cfg["kv_heads"]
    if keys:
        layer["wk"][:32] *= np.float32(1e5)
        for h in range(G):
            layer["wq"][h * D:h * D + 32] = 0.0
    if values:
        last = (cfg["kv_heads"] - 1)
        layer["wv"][last * D + 32:last * D + 64] *= np.float32(1e5)
        for h in range(last * G, (last + 1) * G):
            layer["wo"][:, h * D + 32:h * D + 64] *= np.float32(1e-3)
    for name in ("wq", "wk", "wv", "wo", "gate", "up", "down"):
        layer[name] = (orc.quantize(orc.Q4_0, layer[name]),) + layer[name].shape
    w["head"] = (orc.quantize(orc.Q4_0, w["head"]),) + w["head"].shape
    w["codec"] = orc.Q4_0
    return w


@pytest.mark.parametrize("cfg", [dict(SMALL_Q, layers=1), WIDE_Q], ids=["64", "128"])
@pytest.mark.parametrize("keys,values", [(True, False), (False, True), (True, True)])
def test_rows_beyond_the_range_of_f16(cfg, keys, values):
    w = weights(cfg, keys, values)
    dec, pool, plain = make(cfg, w, 1, et.KV_Q4, False, PAIRS)
    x = plain.norm(w["tok_embd"].astype(np.float64))
    large = np.abs(x @ dense(w["layers"][0]["wv"], orc.Q4_0).T).max(1)
    # attention's output goes on as f16: the first tokens, which attend to few rows, are of moderate values
    small, others = np.flatnonzero(large < 5e4), np.flatnonzero(large > 7e4) if values else np.arange(cfg["vocab"])
    rng = np.random.default_rng(0)
    text = np.concatenate([rng.choice(small, 12), rng.choice(others, 130)])
    seq, before = pool.makeSequence(), 0
    for advance in (20, 1, 64, 50, 1):
        tokens = text[before:before + advance].astype(np.uint32)
        got = dec.execute(pool, [seq], tokens[None])[0]
        want = plain.logits(pool, seq, tokens, before, et.KV_Q4, 2e-3)[-1]
        assert np.abs(got - want).max() <= 2e-3 * np.abs(want).max(), (advance, np.abs(got - want).max() / np.abs(want).max())
        before += advance
    blocks, _ = seq.blocks
    rows = blocks[np.arange(before) // PAGE] * PAGE + np.arange(before) % PAGE
    for which, there in ((0, keys), (1, values)):
        kept = np.abs(pool.read_rows(0, which, rows))
        assert np.isfinite(kept).all() and (kept > 65504).any() == there
