"""How a GGUF file's rope keys become the rotation of a decoder's positions (parsing needs no GPU; loading does)."""
import math
import struct

import numpy as np
import pytest

import effect_torch_b200 as et
from effect_torch_b200.gguf import GgufFile, llama_rope, load_llama_decoder
from oracle import gguf as og

F32 = lambda v: (6, struct.pack("<f", v))
U32 = lambda v: (4, struct.pack("<I", v))
TEXT = lambda v: (8, og.string_value(v))
GEOMETRY = dict(head_dim=64, rope_theta=10000.0)


def rope_of(tmp_path, keys):
    path = tmp_path / "rope.gguf"
    path.write_bytes(og.build([og.metadata_entry(name, *value) for name, value in keys.items()], [], architecture="llama"))
    f = GgufFile(str(path))
    try:
        return llama_rope(f, GEOMETRY, et.INTERLEAVED_PAIRS)
    finally:
        f.close()


@pytest.mark.parametrize("keys,expected", [
    ({}, None),
    ({"llama.rope.dimension_count": U32(64)}, None),
    ({"llama.rope.scaling.type": TEXT("none")}, None),
    ({"llama.rope.scaling.type": TEXT("linear"), "llama.rope.scaling.factor": F32(0.0)}, None),
    ({"llama.rope.dimension_count": U32(32)}, dict(rotary_dim=32)),
    ({"llama.rope.scale_linear": F32(4.0)}, dict(scaling="linear", factor=4.0)),
    ({"llama.rope.scaling.type": TEXT("linear"), "llama.rope.scaling.factor": F32(8.0)}, dict(scaling="linear", factor=8.0)),
    ({"llama.rope.scaling.type": TEXT("yarn"), "llama.rope.scaling.factor": F32(4.0), "llama.rope.scaling.original_context_length": U32(8192)},
     dict(scaling="yarn", factor=4.0, original_context=8192.0)),
    ({"llama.rope.scaling.type": TEXT("yarn"), "llama.rope.scaling.factor": F32(4.0), "llama.context_length": U32(4096), "llama.rope.scaling.yarn_beta_fast": F32(16.0),
      "llama.rope.scaling.attn_factor": F32(2.0)}, dict(scaling="yarn", factor=4.0, original_context=4096.0, beta_fast=16.0, attention_factor=2 * (0.1 * math.log(4.0) + 1)))])
def test_keys_of_a_file(tmp_path, keys, expected):
    config = rope_of(tmp_path, keys)
    if expected is None:
        assert config is None
        return
    want = et.rope_config(64, theta=10000.0, layout=et.INTERLEAVED_PAIRS, **expected)
    for name, _ in et.RopeConfig._fields_:
        assert getattr(config, name) == pytest.approx(getattr(want, name)), name


@pytest.mark.parametrize("keys", [{"llama.rope.scaling.type": TEXT("longrope"), "llama.rope.scaling.factor": F32(4.0)}, {"llama.rope.scaling.type": TEXT("yarn"), "llama.rope.scaling.factor": F32(4.0)}])
def test_what_is_not_known_is_left_out_with_a_warning(tmp_path, keys):
    with pytest.warns(UserWarning, match="positions are not scaled"):
        assert rope_of(tmp_path, keys) is None


@pytest.mark.gpu
def test_a_file_with_scaled_positions_and_frequency_divisors(tmp_path, monkeypatch):
    from tests import helpers, test_gpu_gguf as files
    from tests.gpu_util import runtime

    cfg = helpers.TINY_Q
    weights = helpers.make_weights(cfg, seed=6, codec=2)
    divisors = np.linspace(1, 8, 32).astype(np.float32)
    monkeypatch.setattr(files, "QV", files.QV + [og.metadata_entry("llama.rope.scaling.type", *TEXT("linear")), og.metadata_entry("llama.rope.scaling.factor", *F32(2.0)),
                                                 og.metadata_entry("llama.rope.dimension_count", *U32(64))])
    build = og.build

    def with_divisors(meta, tensors, payloads=None, **kw):
        end = (max(t[3] + t[4] for t in tensors) + 31) // 32 * 32
        payloads["rope_freqs.weight"] = divisors.tobytes()
        return build(meta, tensors + [("rope_freqs.weight", [32], 0, end, 128)], payloads=payloads, **kw)

    monkeypatch.setattr(og, "build", with_divisors)
    path = tmp_path / "scaled.gguf"
    files._llama_file(cfg, weights, path)
    rt = runtime()
    loaded, _ = load_llama_decoder(rt, str(path), batch=2, max_tokens=128, kv_dtype=et.KV_Q4, max_advance=8)
    direct = et.Executable(rt, **{k: cfg[k] for k in ("layers", "d_model", "q_heads", "kv_heads", "head_dim", "ffn", "vocab", "rms_eps")}, batch=2, max_tokens=128,
                           kv_dtype=et.KV_Q4, max_advance=8, rope=et.rope_config(64, theta=cfg["rope_theta"], scaling="linear", factor=2.0), rope_divisors=divisors)
    unscaled = et.Executable(rt, **cfg, batch=2, max_tokens=128, kv_dtype=et.KV_Q4, max_advance=8)
    results = []
    for dec in (loaded, direct, unscaled):
        if dec is not loaded:
            helpers.load_into(dec, weights)
            dec.finalize()
        pool = et.NativeKvPool(rt, cfg["layers"], cfg["kv_heads"], cfg["head_dim"], 128, 16, et.KV_Q4)
        seqs, rng = [pool.makeSequence() for _ in range(2)], np.random.default_rng(3)
        results.append([dec.execute(pool, seqs, rng.integers(0, cfg["vocab"], (2, n)).astype(np.uint32)) for n in (8, 1, 1)])
    for a, b, c in zip(*results):
        np.testing.assert_array_equal(a, b)
        assert not np.array_equal(a, c)
