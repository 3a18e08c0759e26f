"""The 4-bit KV tier: rows into pages and back against the Q4_0 codec (bit exact), attention over them against the same sums in 64 bits.

Tolerance of the decode kernel, with u = 2^-24, A the largest sum |q_d k_d| * scale of a head's tokens and M = sum p |v| / sum p of an output.
A query is held as two f16 numbers, off by 2^-22; the tensor core adds 16 products at a time in f32, which is taken as off by 2^-22 of
the magnitudes added, D / 16 <= 8 times, and the block sums by as many u: a score is off by at most (1 + 8 + 2) 2^-22 A < 2^-18 A and a
weight, relatively, by that and the exponential's 2^-21 (2 ulp and the rounding of its argument). Weights enter sums and their
quotient: twice that. The split weights add 2^-22, the sum over a run of n pages n 2^-22, sums over warps and parts 2^-20.
Weights far below the largest have an absolute error instead: p * dv is held as two f16 numbers after scaling by 2^8 / r, r the power of two at
or above the largest |dv|, so it is off by at most half the smallest f16 step, 2^-25, that is 2^-33 r < 2^-32 max |dv| (which also
covers exponentials that are flushed to 0). A code is at most 8 and max |v| is 7 or 8 max |dv|, so a token adds at most 2^-31.8 max |v| to a
sum that is divided by sum p >= 1: n tokens n 2^-31 max |v|."""
import numpy as np
import pytest
import torch

import effect_torch_b200 as et
import oracle as orc
from tests.gpu_util import dev, empty, host, runtime

pytestmark = pytest.mark.gpu
PAGE = 16


def stored(x):
    """The values that rows of x [..., D] are kept as."""
    flat = np.ascontiguousarray(x, np.float32).reshape(-1, x.shape[-1])
    return orc.dequantize(orc.Q4_0, orc.quantize(orc.Q4_0, flat), *flat.shape).reshape(x.shape)


def lanes_of(rows):
    return dev(np.array(rows, np.int32))


class Cache:
    """Sequences of given lengths over shuffled pages; k and v [kv_heads, length, D] f32 per sequence."""

    def __init__(self, lengths, kv_heads, D, seed=0, spare=3, garbage=False, magnitude=1.0):
        rng = np.random.default_rng(seed)
        self.lengths, self.kv_heads, self.D = lengths, kv_heads, D
        counts = [-(-n // PAGE) for n in lengths]
        pages = sum(counts) + spare
        self.pool = et.NativeKvPool(runtime(), 1, kv_heads, D, pages * PAGE, PAGE, et.KV_Q4)
        order = rng.permutation(pages).astype(np.int32)
        self.first = np.concatenate([[0], np.cumsum(counts)[:-1]]).astype(np.int32)
        self.table = order
        self.tables = dev(order)
        if garbage:  # what pages hold before: scales of infinity
            bad = np.full((1, kv_heads, pages * PAGE, D), np.inf, np.float32)
            runtime().paged_append_into(self.pool, 0, lanes_of([[0, pages * PAGE, 0, 0]]), self.tables, 1, pages * PAGE, dev(bad), dev(bad))
            runtime().synchronize()
        self.k = [rng.normal(size=(kv_heads, n, D)).astype(np.float32) * np.exp(0.5 * rng.normal(size=D)).astype(np.float32) for n in lengths]
        self.v = [magnitude * rng.normal(size=(kv_heads, n, D)).astype(np.float32) for n in lengths]
        for i, n in enumerate(lengths):
            if n:
                runtime().paged_append_into(self.pool, 0, lanes_of([[0, n, 0, self.first[i]]]), self.tables, 1, n, dev(self.k[i][None]), dev(self.v[i][None]))
                runtime().synchronize()

    def rows(self, i):
        at = np.arange(self.lengths[i])
        return self.table[self.first[i] + at // PAGE] * PAGE + at % PAGE


def attend(cache, q, scale, lanes, max_pages, window=None, scratch_fill=None):
    batch, q_heads, D = q.shape
    need = cache.pool.attention_scratch_bytes(batch, q_heads, max_pages)
    scratch = dev(np.full(max(need, 4) // 4, np.nan if scratch_fill is None else scratch_fill, np.float32))
    out = dev(np.full(q.shape, 7.0, np.float32))
    runtime().paged_attention_into(cache.pool, 0, lanes_of(lanes), cache.tables, batch, max_pages, dev(q), q_heads, scale, out, scratch, need, op_window=window)
    return host(out)


def expected(cache, q, scale, lanes, window=None):
    """Results in f64 and how far each may be off."""
    out, room = np.zeros(q.shape), np.zeros(q.shape)
    G = q.shape[1] // cache.kv_heads
    for i, (cursor, advance, start, _) in enumerate(lanes):
        end = cursor + advance
        begin = start if window is None else max(start, end - window, 0)
        if advance == 0 or end <= begin:
            continue
        k, v = (stored(x[i]).astype(np.float64)[:, begin:end] for x in (cache.k, cache.v))
        for h in range(q.shape[1]):
            kk, vv, x = k[h // G], v[h // G], q[i, h].astype(np.float64)
            s = kk @ x * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ vv
            A, M = (np.abs(kk) @ np.abs(x)).max() * abs(scale), w @ np.abs(vv)
            pages = (end - begin) // PAGE + 2
            room[i, h] = (2 * (2.0 ** -18 * A + 2.0 ** -21) + (pages + 5) * 2.0 ** -22) * M + (end - begin) * 2.0 ** -31 * np.nanmax(np.minimum(np.abs(vv), 8 * 65504))
    return out, room


def check(got, want, room):
    fine = np.isfinite(want)  # values beyond the f16 range of the scales (some 5e5) are kept as infinities: their columns have no result
    np.testing.assert_array_equal(np.isfinite(got), fine)
    got, want, room = got[fine], want[fine], room[fine]
    excess = np.max(np.abs(got - want) - room, initial=0.0)
    assert excess <= 0, (excess, np.max(np.abs(got - want)))


@pytest.mark.parametrize("D,block_size,heads", [(32, 1, 1), (32, 3, 2), (64, 16, 2), (96, 4, 3), (96, 5, 1), (128, 16, 8), (128, 32, 1), (160, 16, 2), (256, 8, 1)])
def test_appended_rows_are_q4_0_blocks(D, block_size, heads):
    rng = np.random.default_rng(D + block_size)
    pages, tokens = 24, 2 * block_size + 3
    pool = et.NativeKvPool(runtime(), 2, heads, D, pages * block_size, block_size, et.KV_Q4)
    assert et.pool_state_bytes(2, pages * block_size, heads, D, et.KV_Q4) == 2 * 2 * pages * block_size * heads * D // 32 * 18
    table = rng.permutation(pages).astype(np.int32)
    cursors, advances, first = [0, block_size - 1, 5, 0], [tokens, tokens - 2, 0, 1], [0, 6, 12, 18]
    x = rng.normal(size=(2, 4, heads, tokens, D)).astype(np.float32)
    x[0, 0, 0, 0, :32] = 0.0                       # a block of zeros
    x[1, 0, 0, 1, :32] = np.tile([2.0, -2.0], 16)  # of equal magnitudes the first decides
    x[0, 0, 0, 2, :32] = 1e-30
    x[1, 0, 0, 2, 5] = 1e4
    before = {w: pool.read_rows(1, w, np.arange(pages * block_size)) for w in (0, 1)}
    for offset in (0, 1):  # the second time from rows on an odd 4-byte boundary
        k, v = (dev(np.concatenate([np.zeros(offset, np.float32), s.reshape(-1)])) for s in x)
        runtime().paged_append_into(pool, 1, lanes_of(list(zip(cursors, advances, [0] * 4, first))), dev(table), 4, tokens, k.data_ptr() + 4 * offset, v.data_ptr() + 4 * offset)
        runtime().synchronize()
        for which in (0, 1):
            want = before[which].copy()
            for i in range(4):
                at = cursors[i] + np.arange(advances[i])
                want[table[first[i] + at // block_size] * block_size + at % block_size] = stored(x[which, i, :, :advances[i]]).transpose(1, 0, 2).reshape(advances[i], heads * D)
            rows = np.arange(pages * block_size, dtype=np.uint32)
            np.testing.assert_array_equal(pool.read_rows(1, which, rows).view(np.uint32), want.view(np.uint32))
            out = empty((rows.size * heads * D + 1,))
            for shift in (0, 1):
                runtime().pool_rows_into(pool, 1, which, dev(rows[::-1].astype(np.int32)), rows.size, out.data_ptr() + 4 * shift)
                np.testing.assert_array_equal(host(out)[shift:shift + want.size].view(np.uint32), want[::-1].reshape(-1).view(np.uint32))
            assert not pool.read_rows(0, which, rows).any()  # the other layer


def test_a_nan_takes_no_part_in_its_block():
    pool = et.NativeKvPool(runtime(), 1, 1, 32, 16, 16, et.KV_Q4)
    x = np.linspace(-1, 1, 32, dtype=np.float32).reshape(1, 1, 1, 32)
    x[0, 0, 0, 3] = np.nan
    runtime().paged_append_into(pool, 0, lanes_of([[0, 1, 0, 0]]), dev(np.zeros(1, np.int32)), 1, 1, dev(x), dev(x))
    got = pool.read_rows(0, 0, [0])
    clean = x.copy()
    clean[0, 0, 0, 3] = -1.0  # code 0 of a positive scale is its extreme, here the first value
    np.testing.assert_array_equal(got, stored(clean).reshape(1, -1))


def test_other_tiers_have_device_rows_and_appends_too():
    rng = np.random.default_rng(1)
    for tier, otier in ((et.KV_F32, orc.F32), (et.KV_F16, orc.F16), (et.KV_BF16, orc.BF16), (et.KV_U8, orc.U8)):
        pool = et.NativeKvPool(runtime(), 1, 2, 64, 64, 16, tier)
        x = rng.normal(size=(2, 2, 2, 9, 64)).astype(np.float32)
        table = np.array([3, 1, 0, 2], np.int32)
        runtime().paged_append_into(pool, 0, lanes_of([[10, 9, 0, 0], [0, 4, 0, 2]]), dev(table), 2, 9, dev(x[0]), dev(x[1]))
        runtime().synchronize()
        for which in (0, 1):
            rows = np.array([3 * 16 + 12, 16 + 2, 0, 3, 4], np.uint32)
            want = pool.read_rows(0, which, rows)
            out = empty(want.shape)
            runtime().pool_rows_into(pool, 0, which, dev(rows.astype(np.int32)), 5, out)
            np.testing.assert_array_equal(host(out), want)
            if tier == et.KV_F32:
                np.testing.assert_array_equal(want[0], x[which, 0, :, 2].reshape(-1))
                np.testing.assert_array_equal(want[1], x[which, 0, :, 8].reshape(-1))
                np.testing.assert_array_equal(want[3], x[which, 1, :, 3].reshape(-1))
                assert not want[4].any()


SHAPES = [(1, 1, 64), (4, 2, 64), (3, 1, 128), (8, 2, 128), (5, 1, 128), (14, 2, 64), (8, 1, 128), (9, 1, 128), (24, 2, 64), (16, 1, 128), (32, 2, 128), (32, 8, 128)]


@pytest.mark.parametrize("q_heads,kv_heads,D", SHAPES)
@pytest.mark.parametrize("lengths", [[1], [15, 16, 17], [37, 1, 256, 255], [700, 3, 0, 64, 1500]])
def test_decode_attention(q_heads, kv_heads, D, lengths):
    rng = np.random.default_rng(q_heads + D)
    cache = Cache(lengths, kv_heads, D, seed=len(lengths), garbage=True)
    q = (2 * rng.normal(size=(len(lengths), q_heads, D))).astype(np.float32)
    lanes = [(max(n - 1, 0), min(n, 1), 0, f) for n, f in zip(lengths, cache.first)]
    scale, pages = D ** -0.5, max(1, -(-max(lengths) // PAGE))
    want, room = expected(cache, q, scale, lanes)
    check(attend(cache, q, scale, lanes, pages), want, room)
    # a bound above what lanes attend over changes the plan, not the result
    check(attend(cache, q, scale, lanes, pages + 40), want, room)
    check(attend(cache, q, scale, lanes, 5000), want, room)


@pytest.mark.parametrize("window,starts", [(1, (0, 0)), (5, (0, 0)), (16, (3, 300)), (100, (0, 417)), (None, (1, 400)), (None, (499, 33)), (1000, (500, 500))])
def test_windows_and_starts(window, starts):
    """Rows that a window leaves out, lanes that have nothing left (start at or behind the end), padded lanes."""
    rng = np.random.default_rng(3)
    cache = Cache([500, 420], 2, 64, seed=9, garbage=True)
    q = rng.normal(size=(3, 6, 64)).astype(np.float32)
    lanes = [(499, 1, starts[0], cache.first[0]), (419, 1, min(starts[1], 420), cache.first[1]), (0, 0, 0, 0)]
    for pages in (32, 200):
        got = attend(cache, q, 0.2, lanes, pages, window=window)
        check(got, *expected(cache, q, 0.2, lanes, window))
        assert not got[2].any()


def test_lanes_of_very_different_lengths_and_many_of_them():
    rng = np.random.default_rng(4)
    lengths = [int(n) for n in rng.integers(1, 60, 150)] + [6000, 1, 2500]
    cache = Cache(lengths, 2, 128, seed=5)
    q = rng.normal(size=(len(lengths), 8, 128)).astype(np.float32)
    lanes = [(n - 1, 1, 0, f) for n, f in zip(lengths, cache.first)]
    want, room = expected(cache, q, 0.1, lanes)
    first = attend(cache, q, 0.1, lanes, 375)
    check(first, want, room)
    for fill in (0.0, np.inf):  # nothing is read from scratch that this call did not write, and nothing depends on the run
        np.testing.assert_array_equal(attend(cache, q, 0.1, lanes, 375, scratch_fill=fill).view(np.uint32), first.view(np.uint32))


@pytest.mark.parametrize("magnitude,q_size", [(1e-4, 1e-3), (1e4, 1.0), (1.0, 300.0), (1e-30, 1e-20), (1.0, 0.0)])
def test_magnitudes(magnitude, q_size):
    """Values and queries far from one: powers of two are taken out before anything is held in f16."""
    rng = np.random.default_rng(6)
    cache = Cache([777], 1, 128, seed=7, magnitude=magnitude)
    q = (q_size * rng.normal(size=(1, 4, 128))).astype(np.float32)
    lanes = [(776, 1, 0, 0)]
    check(attend(cache, q, 128 ** -0.5, lanes, 49), *expected(cache, q, 128 ** -0.5, lanes))


def test_growing_scores_and_scales():
    """Every page outdoes the one before, so that references are raised all along."""
    rng = np.random.default_rng(8)
    n = 1200
    cache = Cache([n], 1, 64, seed=8)
    q = np.ones((1, 4, 64), np.float32)
    cache.k[0] = (np.linspace(-8, 8, n)[None, :, None] * np.ones((1, 1, 64)) + 0.01 * rng.normal(size=(1, n, 64))).astype(np.float32)
    cache.v[0] = (2.0 ** (np.arange(n) / 60.0)[None, :, None] * rng.normal(size=(1, n, 64))).astype(np.float32)
    overflows = np.isinf(stored(cache.v[0])).any()
    cache.v[0][..., 32:] *= np.float32(2.0 ** -6)  # this block does not
    assert overflows and np.isfinite(stored(cache.v[0])[..., 32:]).all()
    for a in (0.01, 0.3):
        runtime().paged_append_into(cache.pool, 0, lanes_of([[0, n, 0, 0]]), cache.tables, 1, n, dev(cache.k[0][None]), dev(cache.v[0][None]))
        lanes = [(n - 1, 1, 0, 0)]
        check(attend(cache, q, a, lanes, 75), *expected(cache, q, a, lanes))


def test_a_nan_stays_where_it_is():
    """A NaN in one head's query, an infinity in one lane's values: other heads and lanes are as without."""
    rng = np.random.default_rng(9)
    cache = Cache([300, 200], 2, 64, seed=11)
    q = rng.normal(size=(2, 8, 64)).astype(np.float32)
    lanes = [(299, 1, 0, cache.first[0]), (199, 1, 0, cache.first[1])]
    clean = attend(cache, q, 0.1, lanes, 19)
    q[0, 2, 5] = np.nan
    bad = attend(cache, q, 0.1, lanes, 19)
    assert np.isnan(bad[0, 2]).all()
    keep = np.ones((2, 8), bool)
    keep[0, 2] = False
    np.testing.assert_array_equal(bad[keep], clean[keep])


def test_cursors_beyond_32_bits_of_bytes():
    """Pages whose bytes lie beyond 2^32 of their slab."""
    rng = np.random.default_rng(10)
    kv_heads, D, pages = 8, 128, (1 << 19) + 64
    pool = et.NativeKvPool(runtime(), 1, kv_heads, D, pages * PAGE, PAGE, et.KV_Q4)
    assert (pages - 1) * kv_heads * PAGE * 72 > 1 << 32
    n = 100
    cache = Cache.__new__(Cache)
    cache.lengths, cache.kv_heads, cache.D, cache.pool = [n], kv_heads, D, pool
    cache.table = np.arange(pages - 7, pages, dtype=np.int32)[::-1].copy()
    cache.tables, cache.first = dev(cache.table), [0]
    cache.k, cache.v = ([rng.normal(size=(kv_heads, n, D)).astype(np.float32)] for _ in range(2))
    runtime().paged_append_into(pool, 0, lanes_of([[0, n, 0, 0]]), cache.tables, 1, n, dev(cache.k[0][None]), dev(cache.v[0][None]))
    rows = cache.rows(0)
    out = empty((n, kv_heads * D))
    runtime().pool_rows_into(pool, 0, 0, dev(rows.astype(np.int32)), n, out)
    np.testing.assert_array_equal(host(out), stored(cache.k[0]).transpose(1, 0, 2).reshape(n, -1))
    q = rng.normal(size=(1, 32, D)).astype(np.float32)
    lanes = [(n - 1, 1, 0, 0)]
    check(attend(cache, q, D ** -0.5, lanes, 7), *expected(cache, q, D ** -0.5, lanes))
    check(attend(cache, q, D ** -0.5, lanes, 70), *expected(cache, q, D ** -0.5, lanes))


@pytest.mark.parametrize("D,block_size,q_heads", [(64, 16, 4), (96, 4, 2), (32, 1, 2), (128, 16, 8)])
def test_sequences_over_a_q4_pool(D, block_size, q_heads):
    """The sequence entry points: chunks in reference order (f64), one token by the decode kernel where it serves the geometry."""
    rng = np.random.default_rng(D)
    rt, kv_heads, scale = runtime(), 2, D ** -0.5
    pool = et.NativeKvPool(rt, 1, kv_heads, D, 128, block_size, et.KV_Q4)
    seqs = [pool.makeSequence(), pool.makeSequence()]
    past = [[], []]
    for t in (7, 1, 21, 1, 1):
        q = rng.normal(size=(3, q_heads, t, D)).astype(np.float32)
        k, v = (rng.normal(size=(3, kv_heads, t, D)).astype(np.float32) for _ in range(2))
        for i in range(2):
            past[i].append((stored(k[i]), stored(v[i])))
        out = empty(q.shape)
        decode = block_size == 16 and t == 1 and D in (64, 128)
        if decode:
            rt.kv_attention_decode_into(pool, 0, seqs, 3, 2, dev(q[:, :, 0]), dev(k[:, :, 0]), dev(v[:, :, 0]), q_heads, scale, out=out)
        else:
            rt.kv_attention_into(pool, 0, seqs, 3, 2, t, dev(q), dev(k), dev(v), q_heads, t, scale, out=out)
        got = host(out)
        assert not got[2].any()
        for i in range(2):
            kk, vv = (np.concatenate([p[s] for p in past[i]], axis=1).astype(np.float64) for s in (0, 1))
            n = kk.shape[1]
            for h in range(q_heads):
                g = h // (q_heads // kv_heads)
                s = q[i, h].astype(np.float64) @ kk[g].T * scale
                s[np.triu(np.ones((t, n), bool), n - t + 1)] = -np.inf
                w = np.exp(s - s.max(1, keepdims=True))
                want = w @ vv[g] / w.sum(1, keepdims=True)
                np.testing.assert_allclose(got[i, h], want, rtol=1e-6, atol=3e-5 if decode else 1e-6)  # f32 output; 2^-18 A M is some 3e-5
            seqs[i].commit(np.zeros(t, np.uint32))


def test_a_captured_step_replays():
    """Append and attention of a step in one graph, replayed as the sequence grows; a second graph shares the scratch."""
    rng = np.random.default_rng(12)
    rt, kv_heads, D, q_heads, n = runtime(), 2, 128, 8, 300
    cache = Cache([n + 8], kv_heads, D, seed=13)
    k, v, q = (dev(np.zeros(shape, np.float32)) for shape in ((1, kv_heads, 1, D), (1, kv_heads, 1, D), (1, q_heads, D)))
    lane, out = dev(np.array([[n, 1, 0, 0]], np.int32)), empty((2, 1, q_heads, D))
    need = cache.pool.attention_scratch_bytes(1, q_heads, 20)
    scratch = empty(need // 4)
    stream, graphs = torch.cuda.ExternalStream(rt.stream), []
    for j in range(2):
        graph = torch.cuda.CUDAGraph()
        step = lambda: (rt.paged_append_into(cache.pool, 0, lane, cache.tables, 1, 1, k, v),
                        rt.paged_attention_into(cache.pool, 0, lane, cache.tables, 1, 20, q, q_heads, 0.1, out[j], scratch, need))
        step()
        rt.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step()
        graphs.append(graph)
    for at in (n, n + 1, n + 5):
        x = [rng.normal(size=s.shape).astype(np.float32) for s in (k, v, q)]
        for t, s in zip((k, v, q), x):
            t.copy_(torch.from_numpy(s))
        lane.copy_(torch.tensor([[at, 1, 0, 0]], dtype=torch.int32))
        cache.k[0][:, at], cache.v[0][:, at] = x[0][0, :, 0], x[1][0, :, 0]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for graph in graphs:
                graph.replay()
        got, lanes = host(out), [(at, 1, 0, 0)]
        for j in range(2):
            check(got[j], *expected(cache, x[2], 0.1, lanes))


def test_what_is_refused():
    rt = runtime()
    with pytest.raises(et.BackendError, match="multiple of 32"):
        et.NativeKvPool(rt, 1, 1, 48, 64, 16, et.KV_Q4)
    with pytest.raises(et.BackendError, match="dtype must be"):
        et.NativeKvPool(rt, 1, 1, 64, 64, 16, 5)
    pool = et.NativeKvPool(rt, 1, 2, 64, 64, 16, et.KV_Q4)
    lanes, tables, q, out = lanes_of([[0, 1, 0, 0]]), dev(np.zeros(4, np.int32)), empty((1, 34, 64)), empty((1, 34, 64))
    big = empty(1 << 20)
    for heads, bad in ((3, "grouped-query"), (34, "at most 16")):
        with pytest.raises(et.BackendError, match=bad):
            rt.paged_attention_into(pool, 0, lanes, tables, 1, 4, q, heads, 1.0, out, big, 1 << 20)
        with pytest.raises(et.BackendError, match=bad):
            pool.attention_scratch_bytes(1, heads, 4)
    need = pool.attention_scratch_bytes(1, 4, 100)
    assert need > 0
    with pytest.raises(et.BackendError, match=f"{need} needed"):
        rt.paged_attention_into(pool, 0, lanes, tables, 1, 100, q, 4, 1.0, out, big, need - 1)
    with pytest.raises(et.BackendError, match="needed"):
        rt.paged_attention_into(pool, 0, lanes, tables, 1, 100, q, 4, 1.0, out, None, need)
    for other in (et.NativeKvPool(rt, 1, 2, 96, 64, 16, et.KV_Q4), et.NativeKvPool(rt, 1, 2, 64, 64, 32, et.KV_Q4), et.NativeKvPool(rt, 1, 2, 64, 64, 16, et.KV_F32)):
        with pytest.raises(et.BackendError, match="decode kernel needs"):
            rt.paged_attention_into(other, 0, lanes, tables, 1, 4, q, 4, 1.0, out, big, 1 << 20)
    for call in (lambda: rt.paged_append_into(pool, 1, lanes, tables, 1, 1, q, q), lambda: rt.pool_rows_into(pool, -1, 0, tables, 1, out)):
        with pytest.raises(et.BackendError, match="layer index"):
            call()
    for args in ((lanes, tables, 0, 1, q, q), (lanes, tables, 1, 0, q, q), (lanes, tables, 65536, 1, q, q), (None, tables, 1, 1, q, q), (lanes, tables, 1, 1, None, q)):
        with pytest.raises(et.BackendError, match="kv append"):
            rt.paged_append_into(pool, 0, *args)
    with pytest.raises(et.BackendError, match="which must be"):
        rt.pool_rows_into(pool, 0, 2, tables, 1, out)
    with pytest.raises(et.BackendError, match="number of rows"):
        rt.pool_rows_into(pool, 0, 0, tables, -1, out)
    for tier in (et.KV_Q4, et.KV_F16):
        some = et.NativeKvPool(rt, 1, 2, 64, 64, 16, tier)
        rows = empty((2, 128))
        rt.pool_rows_into(some, 0, 0, dev(np.array([3, 64], np.int32)), 2, rows)
        with pytest.raises(et.BackendError, match=r"row 64 is outside 0\.\.64"):
            rt.synchronize()
        assert not rows.cpu().numpy().any()
    rt.synchronize()


def test_more_rows_than_32_bits_count_are_refused():
    with pytest.raises(et.BackendError, match="at most 2\\^31 - 1 rows"):  # before anything is allocated
        et.NativeKvPool(runtime(), 1, 32, 32, 1 << 26, 16, et.KV_Q4)


@pytest.mark.parametrize("q_heads", [4, 8])
@pytest.mark.parametrize("length", [20, 900])
def test_an_infinite_scale_spoils_its_block_only(q_heads, length):
    """One value beyond the scales' range: the columns of its block have no result, those of the others are as precise as without it."""
    D = 128
    cache = Cache([length], 1, D, seed=5)
    q = np.random.default_rng(7).normal(size=(1, q_heads, D)).astype(np.float32)
    lanes, pages = [(length - 1, 1, 0, cache.first[0])], -(-length // PAGE)
    want, room = expected(cache, q, 0.1, lanes)
    v = cache.v[0].copy()
    v[0, length // 2, 70] = 1e6
    runtime().paged_append_into(cache.pool, 0, lanes_of([[0, length, 0, cache.first[0]]]), cache.tables, 1, length, dev(cache.k[0][None]), dev(v[None]))
    got = attend(cache, q, 0.1, lanes, pages)
    others = np.r_[0:64, 96:128]
    assert not np.isfinite(got[..., 64:96]).any()
    check(got[..., others], want[..., others], room[..., others])
