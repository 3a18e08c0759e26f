"""Bad cached values of one lane and KV head leave every other lane and KV head as they were, bit for bit: runs of work, and the copies ahead of
them, go on across both."""
import numpy as np
import pytest

from tests.gpu_util import dev, runtime
from tests.test_gpu_kv_q4 import PAGE, Cache, attend, lanes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("per_kv", [1, 4, 5, 8, 16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pages", [20, 400])  # the plan of short tables, and runs
@pytest.mark.parametrize("side", ["k", "v"])
def test_bad_values_stay_in_their_lane_and_head(per_kv, D, pages, side):
    rng = np.random.default_rng(per_kv)
    kv_heads, lengths = 2, [300, 200, 310, 1, 17]
    cache = Cache(lengths, kv_heads, D, seed=11)
    q = rng.normal(size=(len(lengths), kv_heads * per_kv, D)).astype(np.float32)
    lanes = [(n - 1, 1, 0, f) for n, f in zip(lengths, cache.first)]
    clean = attend(cache, q, 0.1, lanes, pages)
    assert np.isfinite(clean).all()
    for lane, head, at in ((1, 0, 3), (0, 1, 299), (3, 1, 0)):
        good = {"k": cache.k[lane], "v": cache.v[lane]}
        bad = dict(good, **{side: good[side].copy()})
        bad[side][head, at, 5] = 1e6  # beyond the range of its block's scale
        write = lambda x: runtime().paged_append_into(cache.pool, 0, lanes_of([[0, lengths[lane], 0, cache.first[lane]]]), cache.tables, 1, lengths[lane],
                                                      dev(x["k"][None]), dev(x["v"][None]))
        write(bad)
        got = attend(cache, q, 0.1, lanes, pages)
        hit = np.zeros(clean.shape, bool)
        hit[lane, head * per_kv:(head + 1) * per_kv, :32] = True
        mine = np.zeros(clean.shape, bool)
        mine[lane, head * per_kv:(head + 1) * per_kv] = True
        np.testing.assert_array_equal(got[~mine].view(np.uint32), clean[~mine].view(np.uint32))
        if side == "v":  # a key of infinite scale scores NaN or an infinity, and with -inf its token merely has no weight
            assert not np.isfinite(got[hit]).any() and np.isfinite(got[mine & ~hit]).all()
        write(good)
    np.testing.assert_array_equal(attend(cache, q, 0.1, lanes, pages).view(np.uint32), clean.view(np.uint32))


@pytest.mark.parametrize("per_kv", [4, 8])
@pytest.mark.parametrize("pages", [20, 400])
def test_a_bad_query_stays_in_its_head(per_kv, pages):
    rng = np.random.default_rng(per_kv)
    cache = Cache([300, 200], 2, 64, seed=11)
    q = rng.normal(size=(2, 2 * per_kv, 64)).astype(np.float32)
    lanes = [(299, 1, 0, cache.first[0]), (199, 1, 0, cache.first[1])]
    clean = attend(cache, q, 0.1, lanes, pages)
    for value in (np.nan, np.inf, -np.inf):
        bad = q.copy()
        bad[0, 2, 5] = value
        got = attend(cache, bad, 0.1, lanes, pages)
        keep = np.ones((2, 2 * per_kv), bool)
        keep[0, 2] = False
        np.testing.assert_array_equal(got[keep].view(np.uint32), clean[keep].view(np.uint32))
        assert np.isnan(got[0, 2]).all()
