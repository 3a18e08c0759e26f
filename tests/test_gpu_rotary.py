"""Rotary positions with scaled frequencies against their definition in 64 bits.

Tolerance. With u = 2^-24 and m the attention factor: the reduced angle is exact to f64 but for position * f / pi (2^-52 of some 10^6 half
turns, nothing here), sincospif is within 2 ulp (4 u of a value up to 1), its first-order term within u, the product with m and
its own rounding 2 u, and x cos - y sin adds three roundings of terms up to m (|x| + |y|): in all at most 10 u m (|x| + |y|)."""
import numpy as np
import pytest
import torch

import effect_torch_b200 as et
from tests.gpu_util import dev, empty, host, runtime

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def expected(x, offsets, table):
    """x [batch, heads, steps, head_dim] rotated in f64, and how far each value may be off."""
    f, m = et.rope_frequencies(table.config, None)
    r = table.config.rotary_dim
    position = np.asarray(offsets, np.int64).reshape(-1, 1) + np.arange(x.shape[2])
    angle = (position[..., None].astype(np.longdouble) * f)[:, None]  # [batch or 1, 1, steps, pairs]
    c, s = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    a, b = (slice(0, r // 2), slice(r // 2, r)) if table.config.layout == et.HALF_SPLIT else (slice(0, r, 2), slice(1, r, 2))
    out, room = x.astype(np.float64), np.zeros(x.shape)
    xa, xb = out[..., a].copy(), out[..., b].copy()
    out[..., a], out[..., b] = m * (xa * c - xb * s), m * (xb * c + xa * s)
    room[..., a] = room[..., b] = 10 * U * m * (abs(xa) + abs(xb))
    return out, room


def check(got, want, room):
    worst = np.max(np.abs(got - want) - room)
    assert worst <= 0, worst


RULES = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="llama3", factor=8.0, original_context=8192, theta=500000.0),
         dict(scaling="yarn", factor=32.0, original_context=4096)]


@pytest.mark.parametrize("layout", [et.HALF_SPLIT, et.INTERLEAVED_PAIRS])
@pytest.mark.parametrize("rule", range(len(RULES)))
@pytest.mark.parametrize("head_dim,rotary", [(128, 128), (64, 64), (64, 48), (128, 32), (80, 20), (64, 2), (10, 6), (256, 256), (1024, 1024), (2, 2), (576, 64), (3, 2)])
def test_heads_parts_and_rules(head_dim, rotary, rule, layout):
    rng = np.random.default_rng(head_dim + rotary)
    table = et.RotaryTable(runtime(), head_dim, rotary_dim=rotary, layout=layout, **RULES[rule])
    x = rng.normal(size=(3, 5, 7, head_dim)).astype(np.float32)
    offsets = np.array([0, 131065, 17], np.int64)
    out = empty(x.shape)
    runtime().rotary_into(table, dev(x), dev(offsets), 3, 5, 7, out)
    check(host(out), *expected(x, offsets, table))
    same = dev(x)  # in place, one offset for all
    runtime().rotary_into(table, same, dev(offsets[1:2]), 3, 5, 7, same, n_offsets=1)
    check(host(same), *expected(x, offsets[1:2], table))


@pytest.mark.parametrize("batch,heads,steps", [(1, 1, 1), (1, 40, 1), (32, 40, 1), (2, 3, 1000), (1, 200, 3), (700, 1, 1), (1, 72, 65)])
def test_sizes(batch, heads, steps):
    rng = np.random.default_rng(heads)
    table = et.RotaryTable(runtime(), 128, **RULES[2])
    x = rng.normal(size=(batch, heads, steps, 128)).astype(np.float32)
    offsets = rng.integers(0, 1 << 20, batch)
    out = empty(x.shape)
    runtime().rotary_into(table, dev(x), dev(offsets), batch, heads, steps, out)
    check(host(out), *expected(x, offsets, table))


@pytest.mark.parametrize("layout", [et.HALF_SPLIT, et.INTERLEAVED_PAIRS])
@pytest.mark.parametrize("head_dim,rotary", [(64, 64), (64, 20), (32, 6), (128, 128), (20, 4)])
@pytest.mark.parametrize("batch,heads,steps", [(9001, 1, 1), (3100, 3, 3), (1, 5, 9473), (140, 2, 67), (401, 7, 23), (600, 1, 16)])
def test_several_positions_at_a_time(batch, heads, steps, head_dim, rotary, layout):
    """Many positions of few heads, where a group of positions reaches over one, several or many batch entries."""
    rng = np.random.default_rng(batch + head_dim)
    table = et.RotaryTable(runtime(), head_dim, rotary_dim=rotary, layout=layout, **RULES[2])
    x = rng.normal(size=(batch, heads, steps, head_dim)).astype(np.float32)
    offsets = rng.integers(0, 1 << 17, batch)
    out = empty(x.shape)
    runtime().rotary_into(table, dev(x), dev(offsets), batch, heads, steps, out)
    check(host(out), *expected(x, offsets, table))


@pytest.mark.parametrize("start", [0, 1, 4])
def test_heads_inside_the_rows_of_a_fused_projection(start):
    """q and k heads of [batch, steps, q + 2 kv, D] rows, where the rows start anywhere; v and what lies around stay."""
    rng = np.random.default_rng(start)
    b, t, q, kv, d = 2, 9, 6, 2, 64
    table = et.RotaryTable(runtime(), d, **RULES[3])
    rows = rng.normal(size=start + b * t * (q + 2 * kv) * d + 8).astype(np.float32)
    buffer, offsets = dev(rows), np.array([100, 70000], np.int64)
    strides = (t * (q + 2 * kv) * d, d, (q + 2 * kv) * d)
    x = rows[start:-8].reshape(b, t, q + 2 * kv, d)
    want, room = expected(x[:, :, :q + kv].transpose(0, 2, 1, 3), offsets, table)
    out = empty((b, q + kv, t, d))
    runtime().rotary_into(table, buffer.data_ptr() + 4 * start, dev(offsets), b, q + kv, t, out, x_strides=strides)
    check(host(out), want, room)
    runtime().rotary_into(table, buffer.data_ptr() + 4 * start, dev(offsets), b, q + kv, t, buffer.data_ptr() + 4 * start, x_strides=strides, out_strides=strides)
    after = host(buffer)
    got = after[start:-8].reshape(x.shape)
    check(got[:, :, :q + kv].transpose(0, 2, 1, 3), want, room)
    np.testing.assert_array_equal(got[:, :, q + kv:], x[:, :, q + kv:])
    np.testing.assert_array_equal(after[:start], rows[:start])
    np.testing.assert_array_equal(after[-8:], rows[-8:])


def test_one_head_for_every_query_head():
    """A key head that is repeated (stride 0) on its way."""
    rng = np.random.default_rng(3)
    table = et.RotaryTable(runtime(), 64)
    x = rng.normal(size=(2, 1, 4, 64)).astype(np.float32)
    out = empty((2, 5, 4, 64))
    runtime().rotary_into(table, dev(x), dev(np.array([3, 4], np.int64)), 2, 5, 4, out, x_strides=(4 * 64, 0, 64))
    check(host(out), *expected(np.repeat(x, 5, axis=1), [3, 4], table))


def test_passed_values_are_copied_bit_for_bit_and_far_positions_hold():
    table = et.RotaryTable(runtime(), 64, rotary_dim=32)
    x = np.random.default_rng(4).normal(size=(2, 3, 1, 64)).astype(np.float32)
    x[0, 0, 0, 40:44] = [np.inf, -np.inf, np.nan, -0.0]
    offsets = np.array([(1 << 33) + 5, -(1 << 20)], np.int64)
    out = empty(x.shape)
    runtime().rotary_into(table, dev(x), dev(offsets), 2, 3, 1, out)
    got = host(out)
    np.testing.assert_array_equal(got[..., 32:].view(np.uint32), x[..., 32:].view(np.uint32))
    want, room = expected(x, offsets, table)
    # 2^33 positions: position * f / pi is off by 2^-53 of 2.7e9 half turns, pi times that is 1e-6
    check(got[..., :32], want[..., :32], room[..., :32] + 1e-6 * 4 * np.abs(x[..., :32]).max())


def test_a_captured_call_replays_on_new_positions():
    rng = np.random.default_rng(5)
    rt, table = runtime(), et.RotaryTable(runtime(), 128, **RULES[3])
    x, offsets, out = dev(np.zeros((4, 6, 1, 128), np.float32)), dev(np.zeros(4, np.int64)), empty((4, 6, 1, 128))
    call = lambda: rt.rotary_into(table, x, offsets, 4, 6, 1, out)
    call()
    rt.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.ExternalStream(rt.stream)
    with torch.cuda.graph(graph, stream=stream):
        call()
    values, at = rng.normal(size=(4, 6, 1, 128)).astype(np.float32), rng.integers(0, 1 << 17, 4)
    x.copy_(torch.from_numpy(values))
    offsets.copy_(torch.from_numpy(at))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.replay()
    check(host(out), *expected(values, at, table))


def test_what_is_refused():
    rt, table = runtime(), et.RotaryTable(runtime(), 64)
    x, o, out = empty((2, 3, 4, 64)), dev(np.zeros(2, np.int64)), empty((2, 3, 4, 64))
    for args, kw, message in [((x, o, 2, 3, 4, out), dict(n_offsets=3), "3 offsets for batch 2"), ((x, o, -1, 3, 4, out), {}, "negative sizes"),
                              ((None, o, 2, 3, 4, out), {}, "device buffers"), ((x, None, 2, 3, 4, out), {}, "device buffers"),
                              ((x, o, 2, 3, 4, out), dict(x_strides=(-1, 64, 64)), "strides"), ((x, o, 2, 3, 4, out), dict(out_strides=(768, 256, 63)), "strides"),
                              ((x, o, 2, 3, 4, out), dict(out_strides=(1 << 62, 256, 64)), "strides"),
                              ((x, o, 2, 3, 4, x), dict(out_strides=(768, 64, 192)), "in place"), ((x, o, 2, (1 << 20) + 1, 4, out), {}, "2\\^20 heads"),
                              ((x, o, 2, 3, 1 << 31, out), {}, "2\\^20 heads")]:
        with pytest.raises(et.BackendError, match=message):
            rt.rotary_into(table, *args, **kw)
    rt.rotary_into(table, x, o, 2, 0, 4, out)
    with pytest.raises(et.BackendError, match="rotated part"):
        et.RotaryTable(rt, 64, rotary_dim=65)
    other = et.Runtime(0)
    with pytest.raises(et.BackendError, match="different runtime"):
        other.rotary_into(table, x, o, 2, 3, 4, out)
    other.close()
    table.close()
    with pytest.raises(et.BackendError, match="different runtime"):
        rt.rotary_into(table, x, o, 2, 3, 4, out)
