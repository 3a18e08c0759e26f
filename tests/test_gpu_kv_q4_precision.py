"""How closely decode attention over the 4-bit tier follows the stored values where their sizes differ widely: blocks of a head, tokens of very
little weight, rows far larger than the others.

Tolerance, with A, M and the pages' term as in test_gpu_kv_q4.py: (2 (2^-18 A + 2^-21) + (pages + 5) 2^-22) M for the scores, exponentials, the
products held in 22 bits (2^-22, within the pages' term) and the sums, relative to M = sum w |v| of the column itself. On top a product w dv
below the range of its f16 numbers is off by at most half their smallest step, 2^-25, in units in which the largest product w max_b dv of
a token (w its part of the sum of the weights, W the largest such product) is at least 2^10.9: a head's reference is set so that it is 2^11, by
a logarithm that is at most 0.09 too large. Times a code of at most 8 that is 2^-32.9 W a token, taken as 2^-32.5; up to four heads per KV head hold
the second number times 2^11, so 2^-43.5. Scales below 2^-14 count as 2^-14 in W, where that logarithm is not taken of the value."""
import numpy as np
import pytest

import oracle as orc
from tests.gpu_util import dev, runtime
from tests.test_gpu_kv_q4 import PAGE, Cache, attend, lanes_of, stored

pytestmark = pytest.mark.gpu


def scales(x):
    """Largest |block scale| of each row of x [..., D]."""
    flat = np.ascontiguousarray(x, np.float32).reshape(-1, x.shape[-1])
    packed = np.frombuffer(np.ascontiguousarray(orc.quantize(orc.Q4_0, flat)).tobytes(), np.uint8).reshape(flat.shape[0], -1, 18)
    return np.abs(packed[:, :, :2].copy().view(np.float16)[..., 0]).astype(np.float64).max(1).reshape(x.shape[:-1])


def expected(k, v, q, scale):
    """Of one lane: k, v [kv_heads, n, D], q [q_heads, D]."""
    out, room = np.zeros(q.shape), np.zeros(q.shape)
    G = q.shape[0] // len(k)
    kk, vv, dv = stored(k).astype(np.float64), stored(v).astype(np.float64), scales(v)
    dv = np.maximum(np.where(np.isinf(dv), 0.0, dv), 2.0 ** -14)
    floor = 2.0 ** -(43.5 if G <= 4 else 32.5)
    for h in range(q.shape[0]):
        key, value, x = kk[h // G], vv[h // G], q[h].astype(np.float64)
        s = key @ x * scale
        w = np.exp(s - s.max())
        w /= w.sum()
        with np.errstate(invalid="ignore"):
            out[h] = w @ value
        A, M = (np.abs(key) @ np.abs(x)).max() * abs(scale), w @ np.abs(value)
        room[h] = (2 * (2.0 ** -18 * A + 2.0 ** -21) + (key.shape[0] // PAGE + 7) * 2.0 ** -22) * M + key.shape[0] * floor * (w * dv[h // G]).max()
    return out, room


def check(k, v, q, scale):
    n = k.shape[1]
    cache = Cache([1], k.shape[0], k.shape[2], spare=-(-n // PAGE) + 2)  # its pages are overwritten
    runtime().paged_append_into(cache.pool, 0, lanes_of([[0, n, 0, 0]]), cache.tables, 1, n, dev(k[None]), dev(v[None]))
    runtime().synchronize()
    want, room = expected(k, v, q, scale)
    pages = -(-n // PAGE)
    for bound in (pages, pages + 40):
        got = attend(cache, q[None], scale, [(n - 1, 1, 0, 0)], bound)[0]
        fine = np.isfinite(want)  # values beyond 8 * 65504 are kept as infinities: the columns of their blocks have no result
        np.testing.assert_array_equal(np.isfinite(got), fine)
        excess = np.where(fine, np.abs(got - np.where(fine, want, 0.0)) / room, 0.0)
        assert excess.max() <= 1, (bound, excess.max(), np.unravel_index(excess.argmax(), excess.shape))


HEADS = [(1, 1), (4, 1), (8, 2), (5, 1), (8, 1), (16, 1)]


@pytest.mark.parametrize("q_heads,kv_heads", HEADS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 3, 40, 700])
def test_blocks_of_very_different_sizes(q_heads, kv_heads, D, n):
    """Blocks of a head up to 2e4 apart: each block's columns are as precise as if it were alone."""
    rng = np.random.default_rng(n + q_heads)
    k, v = (rng.normal(size=(kv_heads, n, D)).astype(np.float32) for _ in range(2))
    sizes = np.array([3000.0, 0.15, 40.0, 1.0])[:D // 32]
    v *= np.repeat(sizes, 32).astype(np.float32)
    check(k, v, rng.normal(size=(q_heads, D)).astype(np.float32), 0.1)


@pytest.mark.parametrize("q_heads,kv_heads", HEADS[:3])
@pytest.mark.parametrize("n", [1, 40, 700])
def test_blocks_a_million_apart(q_heads, kv_heads, n):
    rng = np.random.default_rng(n)
    k, v = (rng.normal(size=(kv_heads, n, 128)).astype(np.float32) for _ in range(2))
    v *= np.repeat(np.array([1e5, 0.1, 1e5, 3.0]), 32).astype(np.float32)
    check(k, v, rng.normal(size=(q_heads, 128)).astype(np.float32), 0.1)


@pytest.mark.parametrize("q_heads,kv_heads", HEADS)
@pytest.mark.parametrize("n", [400, 30000])
def test_one_token_draws_nearly_all_weight_and_has_small_values(q_heads, kv_heads, n):
    """The others weigh some 2^-28 each, are alike, and make the result: what each of them is off by adds up."""
    rng = np.random.default_rng(n)
    D = 64
    k, v = np.zeros((kv_heads, n, D), np.float32), np.zeros((kv_heads, n, D), np.float32)
    k[..., 0], k[:, 0, 0] = -1.0, 1.0
    v[:, 1:] = rng.normal(size=(kv_heads, 1, D))
    v[:, 0] = 1e-4 * rng.normal(size=(kv_heads, D))
    q = np.zeros((q_heads, D), np.float32)
    q[:, 0] = np.linspace(9.0, 10.0, q_heads)
    check(k, v, q, 1.0)


@pytest.mark.parametrize("q_heads,kv_heads", HEADS)
@pytest.mark.parametrize("at,size", [(0, 2e5), (50, 2e5), (599, 2e5), (0, 1e5), (50, 1e5), (599, 1e5)])
def test_an_outsized_row_of_no_weight(q_heads, kv_heads, at, size):
    """One row of values 1e5 times the others', whose weight makes it the smaller part of the sum; with 2e5 it leaves the range that scales
    have in some blocks."""
    rng = np.random.default_rng(at)
    n, D = 600, 128
    k, v = (rng.normal(size=(kv_heads, n, D)).astype(np.float32) for _ in range(2))
    q = 0.1 * rng.normal(size=(q_heads, D)).astype(np.float32)
    q[:, 0], k[:, :, 0], k[:, at, 0] = 12.0, 1.0, -1.0
    v[:, at] *= size
    check(k, v, q, 0.7)


@pytest.mark.parametrize("q_heads", [4, 8])
def test_scales_below_the_normal_range_of_f16(q_heads):
    rng = np.random.default_rng(3)
    k, v = (rng.normal(size=(1, 300, 128)).astype(np.float32) for _ in range(2))
    check(k, v * np.float32(2e-6), rng.normal(size=(q_heads, 128)).astype(np.float32), 0.1)
    v[..., 32:] *= np.float32(1e-5)
    check(k, v, rng.normal(size=(q_heads, 128)).astype(np.float32), 0.1)


@pytest.mark.parametrize("q_heads", [1, 4, 8])
@pytest.mark.parametrize("power", [10, 20, 22, 23, 24, 25, 26, 27, 28, 29, 31, 40, 60])
@pytest.mark.parametrize("size", [1e-5, 1.0, 1e4])
def test_scores_beyond_what_f32_resolves(q_heads, power, size):
    """Scores of some 2^power that differ by a few units, or by what f32 keeps of them there: whatever the weights, a result is a mean of the
    values, within a part in 2^18 of the largest (two splits and the sums' own roundings)."""
    rng = np.random.default_rng(power)
    n, D = 700, 64
    k, v = np.zeros((1, n, D), np.float32), (size * np.exp(rng.normal(size=(1, n, 1))) * rng.normal(size=(1, n, D))).astype(np.float32)
    k[..., 0], k[..., 32] = 1.0, rng.normal(size=n)
    q = np.zeros((1, q_heads, D), np.float32)
    q[..., 0], q[..., 32] = 2.0 ** power * 0.7, 20.0
    cache = Cache([1], 1, D, spare=-(-n // PAGE) + 2)
    runtime().paged_append_into(cache.pool, 0, lanes_of([[0, n, 0, 0]]), cache.tables, 1, n, dev(k[None].reshape(1, 1, n, D)), dev(v[None].reshape(1, 1, n, D)))
    values = stored(v)[0]
    fine = np.isfinite(values).all(0)  # with 1e4 some values leave the range that scales have: the columns of their blocks have no result
    assert size == 1e4 or fine.all()
    values = values[:, fine]
    room = 2.0 ** -18 * np.abs(values).max(initial=0.0)
    for pages in (44, 100):
        got = attend(cache, q, 1.0, [(n - 1, 1, 0, 0)], pages)[0]
        np.testing.assert_array_equal(np.isfinite(got), np.broadcast_to(fine, got.shape))
        got = got[:, fine]
        assert (got >= values.min(0) - room).all() and (got <= values.max(0) + room).all()
