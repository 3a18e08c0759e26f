"""What the operators of long contexts say when they refuse a call, and what calls that are served must not take."""
import numpy as np
import pytest

import effect_torch_b200 as et
from tests.gpu_util import dev, empty, runtime

pytestmark = pytest.mark.gpu


def test_the_decode_kernels_name_the_tiers_they_take():
    rt = runtime()
    lanes, tables, q, out = dev(np.array([[0, 1, 0, 0]], np.int32)), dev(np.zeros(4, np.int32)), empty((1, 4, 64)), empty((1, 4, 64))
    pool = et.NativeKvPool(rt, 1, 2, 64, 64, 16, et.KV_F32)
    with pytest.raises(et.BackendError, match="needs an f16, bf16, u8 or q4 pool with 16-token pages"):
        rt.paged_attention_into(pool, 0, lanes, tables, 1, 4, q, 4, 1.0, out, empty(1 << 20), 1 << 20)
    for tier in (et.KV_F16, et.KV_BF16, et.KV_U8, et.KV_Q4):
        et.NativeKvPool(rt, 1, 2, 64, 64, 16, tier).attention_scratch_bytes(1, 4, 4)
