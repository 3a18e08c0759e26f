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


@pytest.mark.parametrize("exact", [True, False])
def test_scoring_token_by_token_holds_no_logits_of_its_own(exact):
    import oracle as orc
    from tests import helpers
    from tests.test_gpu_long_context import SMALL, SMALL_Q, make

    cfg = SMALL if exact else SMALL_Q
    dec, pool, _ = make(cfg, helpers.make_weights(cfg, seed=1, codec=0 if exact else orc.Q4_0), 4, et.KV_F16, exact, None)
    seqs, rt = [pool.makeSequence() for _ in range(4)], runtime()
    before = rt.memory_bytes
    first = dec.score(pool, seqs, np.ones((4, 1)), np.full((4, 1), 5), top=2)
    assert rt.memory_bytes - before < 4 * cfg["vocab"]  # less than a row of logits
    dec.score(pool, seqs, np.ones((4, 3)), np.ones((4, 3)), top=2)
    assert rt.memory_bytes - before > 12 * 4 * cfg["vocab"]
    again = [pool.makeSequence() for _ in range(4)]
    for a, b in zip(first, dec.score(pool, again, np.ones((4, 1)), np.full((4, 1), 5), top=2)):
        np.testing.assert_array_equal(a, b)


def test_scores_of_a_part_of_the_vocabulary_are_refused():
    """Also where the decoder of that part stands alone: its logits are no distribution."""
    from tests import helpers
    from tests.test_gpu_long_context import SMALL

    half = dict(SMALL, vocab=750)
    w = helpers.make_weights(SMALL, seed=1)
    for first, whole in ((0, False), (750, False), (0, True)):
        cfg = SMALL if whole else half
        dec = et.Executable(runtime(), **cfg, batch=1, max_tokens=64, exact=True, vocab_global=1500, head_first_row=first)
        helpers.load_into(dec, dict(w, head=w["head"][first:first + cfg["vocab"]]))
        dec.finalize()
        pool = et.NativeKvPool(runtime(), cfg["layers"], cfg["kv_heads"], cfg["head_dim"], 64, 16, et.KV_F32)
        seqs = [pool.makeSequence()]
        if whole:
            dec.score(pool, seqs, [[3]], [[4]])
            continue
        with pytest.raises(et.BackendError, match="vocabulary-parallel head"):
            dec.score(pool, seqs, [[3]], [[4]])
        assert seqs[0].cursor == 0
        dec.execute(pool, seqs, [[3]])


@pytest.mark.parametrize("tier", [et.KV_F16, et.KV_U8, et.KV_Q4])
def test_scratch_between_floats_is_refused(tier):
    """Scratch is given in bytes, so that it may begin anywhere; partial sums in it are floats."""
    rt = runtime()
    pool = et.NativeKvPool(rt, 1, 2, 64, 64, 16, tier)
    lanes, tables, q, out = dev(np.array([[0, 1, 0, 0]], np.int32)), dev(np.zeros(4, np.int32)), empty((1, 4, 64)), empty((1, 4, 64))
    pages = 400
    need = pool.attention_scratch_bytes(1, 4, pages)
    assert need > 0
    scratch = empty(need // 4 + 8)
    for shift in (1, 2, 3):
        with pytest.raises(et.BackendError, match="scratch must lie on a 4-byte boundary"):
            rt.paged_attention_into(pool, 0, lanes, tables, 1, pages, q, 4, 1.0, out, scratch.data_ptr() + shift, need + 8)
    rt.paged_append_into(pool, 0, lanes, tables, 1, 1, dev(np.ones((1, 2, 1, 64), np.float32)), dev(np.full((1, 2, 1, 64), 0.5, np.float32)))
    rt.paged_attention_into(pool, 0, lanes, tables, 1, pages, q, 4, 1.0, out, scratch.data_ptr() + 4, need + 4)
    rt.synchronize()
    assert np.isfinite(out.cpu().numpy()).all()
