"""GGUF files whose rope keys or divisors no rotation has: they load, as before such keys were read, and say so (no GPU needed)."""
import warnings

import numpy as np
import pytest

import effect_torch_b200 as et
from effect_torch_b200.gguf import GgufFile, llama_rope_divisors
from oracle import gguf as og
from tests.test_gguf_rope import F32, TEXT, U32, rope_of

LINEAR = {"llama.rope.scaling.type": TEXT("linear")}
YARN = {"llama.rope.scaling.type": TEXT("yarn"), "llama.rope.scaling.factor": F32(4.0), "llama.rope.scaling.original_context_length": U32(8192)}


@pytest.mark.parametrize("keys", [dict(LINEAR, **{"llama.rope.scaling.factor": F32(0.5)}), dict(LINEAR, **{"llama.rope.scaling.factor": F32(-2.0)}),
                                  dict(LINEAR, **{"llama.rope.scaling.factor": F32(float("nan"))}), {"llama.rope.dimension_count": U32(0)},
                                  {"llama.rope.dimension_count": U32(63)}, {"llama.rope.dimension_count": U32(128)}, dict(YARN, **{"llama.rope.scaling.yarn_beta_fast": F32(0.5)}),
                                  dict(YARN, **{"llama.rope.scaling.factor": F32(0.25)}), dict(YARN, **{"llama.rope.scaling.attn_factor": F32(-1.0)}),
                                  dict(YARN, **{"llama.rope.scaling.attn_factor": F32(2.0), "llama.rope.scaling.factor": F32(-4.0)})])
def test_keys_that_cannot_be_followed(tmp_path, keys):
    with pytest.warns(UserWarning, match="rope keys cannot be followed.*positions are not scaled"):
        assert rope_of(tmp_path, keys) is None


def test_keys_that_can_be_followed_give_no_warning(tmp_path):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert rope_of(tmp_path, YARN).scaling == et.ROPE_SCALINGS["yarn"]
        assert rope_of(tmp_path, {"llama.rope.dimension_count": U32(2)}).rotary_dim == 2


def divisors_of(tmp_path, values, pairs, codec=0):
    payload = np.asarray(values, np.float32).tobytes()
    path = tmp_path / "divisors.gguf"
    tensors = [] if values is None else [("rope_freqs.weight", [len(values)], codec, 0, len(payload))]
    path.write_bytes(og.build([], tensors, payloads={} if values is None else {"rope_freqs.weight": payload}, architecture="llama"))
    f = GgufFile(str(path))
    try:
        return llama_rope_divisors(f, pairs)
    finally:
        f.close()


def test_divisors_of_a_file(tmp_path):
    values = np.linspace(1, 8, 32).astype(np.float32)
    np.testing.assert_array_equal(divisors_of(tmp_path, values, 32), values)
    assert divisors_of(tmp_path, None, 32) is None
    for bad in (values[:31], np.where(np.arange(32) == 3, 0, values), np.where(np.arange(32) == 31, np.nan, values), -values):
        with pytest.warns(UserWarning, match="does not hold 32 positive F32 divisors"):
            assert divisors_of(tmp_path, bad, 32) is None


@pytest.mark.parametrize("keys,factor", [({"llama.rope.scaling.factor": F32(4.0)}, 4.0), ({"llama.rope.scaling.factor": F32(4.0), "llama.rope.scale_linear": F32(2.0)}, 4.0),
                                         ({"llama.rope.scaling.factor": F32(1.0)}, None), ({"llama.rope.scaling.factor": F32(0.0)}, None),
                                         ({"llama.rope.scaling.type": TEXT("none"), "llama.rope.scaling.factor": F32(4.0)}, None)])
def test_a_factor_without_a_type_is_linear(tmp_path, keys, factor):
    config = rope_of(tmp_path, keys)
    assert (config is None) == (factor is None)
    assert config is None or (config.scaling, config.factor) == (et.ROPE_SCALINGS["linear"], factor)
