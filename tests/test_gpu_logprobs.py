"""Log probabilities of given tokens, entropy and alternatives against their definitions in 64 bits.

Tolerances. Values are f32, sums of at most a few hundred values are f32, the rest f64, so with u = 2^-24 and d = x - m (f32, |d| <= 200):
an exponential is off by the rounding of d (u |d|), of d * log2 e and by ex2.approx (2 ulp), in all (2 |d| + 4) u relative. Terms beyond
|d| = 16 weigh nothing at 2^-24, so s and its logarithm are off by at most (2 * 16 + 4) u and 256 additions in pairs and in sequence
(at most 256 u, in practice some tens): |error of ln s| <= 300 u = 1.8e-5, and a log probability adds its own rounding, u |lp|.
t / s is a mean of d under the same weights: twice that times its size."""
import numpy as np
import pytest
import torch

import effect_torch_b200 as et
from tests.gpu_util import dev, empty, host, runtime

pytestmark = pytest.mark.gpu
ABS = 300 * 2.0 ** -24
REL = 2.0 ** -23


def expected(logits, targets, top):
    """Per row in f64: log probability, entropy, first tokens by (value descending, token ascending) and their log probabilities."""
    x = logits.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(1, keepdims=True)
        e = np.exp(x - m)
        lp = (x - m) - np.log(e.sum(1, keepdims=True))  # not x - (m + ln s): 64 bits do not hold 3.4e38 + 4
        p = np.exp(lp)
        entropy = -np.where(p > 0, p * lp, np.where(np.isnan(p), np.nan, 0.0)).sum(1)
    order = np.argsort(-logits, axis=1, kind="stable")[:, :top]
    return lp[np.arange(len(x)), targets], entropy, order, np.take_along_axis(lp, order, 1)


def score(logits, targets, top, stride=None, offset=0):
    rows, vocab = logits.shape
    stride = vocab if stride is None else stride
    buffer = np.full(offset + rows * stride + 8, np.nan, np.float32)  # what lies between and around the rows is never part of one
    for r in range(rows):
        buffer[offset + r * stride:offset + r * stride + vocab] = logits[r]
    x = dev(buffer)
    lp, entropy = empty(rows), empty(rows)
    tokens, alternatives = empty((rows, top), torch.int32), empty((rows, top))
    runtime().logprobs_into(x.data_ptr() + 4 * offset, rows, vocab, dev(targets.astype(np.int32)), lp, entropy, top, tokens, alternatives, row_stride=stride)
    return host(lp), host(entropy), host(tokens), host(alternatives)


def check(logits, targets, top, **layout):
    got, want = score(logits, targets, top, **layout), expected(logits, targets, top)
    np.testing.assert_allclose(got[0], want[0], rtol=REL, atol=ABS)
    np.testing.assert_allclose(got[1], want[1], rtol=REL, atol=ABS + 2 * ABS * np.nanmax(np.abs(want[1]), initial=1.0))
    np.testing.assert_array_equal(got[2], want[2])
    np.testing.assert_allclose(got[3], want[3], rtol=REL, atol=ABS)


@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (2, 31, 31), (5, 33, 32), (1, 127, 5), (7, 1000, 20), (2, 2047, 32), (4, 2048, 1),
                                            (3, 4096, 20), (2, 50257, 32), (1, 128256, 20), (32, 128256, 5), (300, 128256, 0), (300, 4099, 3), (1, 200003, 32)])
def test_rows_of_all_lengths(rows, vocab, top):
    rng = np.random.default_rng(rows * 1000003 + vocab + top)
    logits = (rng.normal(size=(rows, vocab)) * 2.5).astype(np.float32)
    check(logits, rng.integers(0, vocab, rows), top)


@pytest.mark.parametrize("offset,stride", [(0, 1001), (1, 1000), (2, 1003), (3, 1007), (1, 4096)])
def test_rows_that_start_on_any_boundary(offset, stride):
    rng = np.random.default_rng(offset)
    check(rng.normal(size=(6, 1000)).astype(np.float32), rng.integers(0, 1000, 6), 8, stride=stride, offset=offset)


@pytest.mark.parametrize("vocab", [70, 3000, 128256])
def test_ties_go_to_the_lower_token(vocab):
    rng = np.random.default_rng(vocab)
    logits = np.stack([np.zeros(vocab), rng.integers(-2, 3, vocab), np.arange(vocab) // 40 % 7, -np.arange(vocab) / 64.0, np.arange(vocab) / 64.0,
                       np.where(rng.random(vocab) < 0.5, 0.0, -0.0)]).astype(np.float32)
    check(logits, rng.integers(0, vocab, len(logits)), 32)


def test_an_order_that_overflows_the_list_of_candidates():
    """Values that fall with their token's piece of 2048, so that few threads hold everything large."""
    vocab = 128256
    piece, within = np.arange(vocab) // 2048, np.arange(vocab) % 2048
    logits = np.where(within < 128, 50.0 - 0.001 * within - 0.01 * piece, -within / 100.0).astype(np.float32)[None]
    check(logits, np.array([77]), 32)
    many = np.where(within < 128, 10.0, np.float32(-1.0)).astype(np.float32)[None]
    check(many, np.array([2048]), 32)


@pytest.mark.parametrize("vocab", [50, 5000, 128256])
def test_barred_tokens_and_lowest_values(vocab):
    rng = np.random.default_rng(vocab + 1)
    logits = rng.normal(size=(6, vocab)).astype(np.float32)
    logits[0, rng.random(vocab) < 0.9] = -np.inf
    logits[1, :] = -np.inf
    logits[1, 17] = 3.0                                      # one token left
    logits[2, :-1] = np.finfo(np.float32).min                # masked by the lowest value
    logits[3, :] = np.finfo(np.float32).min                  # everything masked by it: even chances
    logits[4, :] = -np.inf                                   # everything barred: no distribution
    logits[5, ::2] = 60000.0
    targets = np.array([int(np.argmax(logits[0])), 17, vocab - 1, 5, 6, 1])
    check(logits, targets, min(vocab, 32))
    assert np.isneginf(score(logits[1:2], np.array([18]), 3)[0][0])


def test_outputs_that_are_not_asked_for():
    rng = np.random.default_rng(5)
    logits, targets = rng.normal(size=(4, 700)).astype(np.float32), rng.integers(0, 700, 4)
    want = expected(logits, targets, 3)
    x, rt = dev(logits), runtime()
    lp, entropy, tokens, alternatives = empty(4), empty(4), empty((4, 3), torch.int32), empty((4, 3))
    rt.logprobs_into(x, 4, 700, dev(targets.astype(np.int32)), lp)
    np.testing.assert_allclose(host(lp), want[0], rtol=REL, atol=ABS)
    rt.logprobs_into(x, 4, 700, entropy=entropy)
    np.testing.assert_allclose(host(entropy), want[1], rtol=REL, atol=8 * ABS)
    rt.logprobs_into(x, 4, 700, top=3, top_tokens=tokens, top_logprobs=alternatives)
    np.testing.assert_array_equal(host(tokens), want[2])
    rt.logprobs_into(x, 4, 700)
    rt.logprobs_into(x, 0, 700, dev(targets.astype(np.int32)), lp)


def test_results_do_not_depend_on_the_run():
    rng = np.random.default_rng(6)
    logits, targets = rng.normal(size=(9, 128256)).astype(np.float32), rng.integers(0, 128256, 9)
    first = score(logits, targets, 32)
    for _ in range(3):
        for a, b in zip(first, score(logits, targets, 32)):
            np.testing.assert_array_equal(a.view(np.uint32), b.view(np.uint32))


def test_a_captured_call_replays_on_new_logits():
    rng = np.random.default_rng(7)
    rt, rows, vocab = runtime(), 3, 9001
    x, t = dev(np.zeros((rows, vocab), np.float32)), dev(np.zeros(rows, np.int32))
    lp, entropy, tokens, alternatives = empty(rows), empty(rows), empty((rows, 4), torch.int32), empty((rows, 4))
    call = lambda: rt.logprobs_into(x, rows, vocab, t, lp, entropy, 4, tokens, alternatives)
    call()
    rt.synchronize()
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.ExternalStream(rt.stream)
    with torch.cuda.graph(graph, stream=stream):
        call()
    for _ in range(2):
        logits, targets = rng.normal(size=(rows, vocab)).astype(np.float32), rng.integers(0, vocab, rows).astype(np.int32)
        x.copy_(torch.from_numpy(logits))
        t.copy_(torch.from_numpy(targets))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        want = expected(logits, targets, 4)
        np.testing.assert_allclose(host(lp), want[0], rtol=REL, atol=ABS)
        np.testing.assert_array_equal(host(tokens), want[2])


def test_what_is_refused_or_reported():
    rt = runtime()
    x, t, f = dev(np.zeros((2, 40), np.float32)), dev(np.zeros(2, np.int32)), empty(64)
    i = empty(64, torch.int32)
    for args, message in [((x, 2, 0), "must be non-empty"), ((x, 2, 1048577), "exceeds limit"), ((x, -1, 40), "number of rows"),
                          ((x, 2, 40, t, f, None, 33, i, f), r"must be in \[0, 32\]"), ((x, 2, 40, t, f, None, -1, i, f), r"must be in \[0, 32\]"),
                          ((x, 2, 5, t, f, None, 6, i, f), r"must be in \[0, 5\]"), ((x, 2, 40, t, None), "must be device buffers"),
                          ((x, 2, 40, None, f), "must be device buffers"), ((None, 2, 40, t, f), "must be device buffers"),
                          ((x, 2, 40, t, f, None, 2, None, f), "must be device buffers")]:
        with pytest.raises(et.BackendError, match=message):
            rt.logprobs_into(*args)
    with pytest.raises(et.BackendError, match="shorter than a row"):
        rt.logprobs_into(x, 2, 40, t, f, row_stride=39)
    with pytest.raises(et.BackendError, match="overflow"):
        rt.logprobs_into(x, 4, 40, t, f, row_stride=1 << 61)
    rt.logprobs_into(x, 2, 40, dev(np.array([1, 40], np.int32)), f)
    with pytest.raises(et.BackendError, match=r"target 40 is outside 0\.\.40"):
        rt.synchronize()
    assert np.isnan(f.cpu().numpy()[1]) and abs(f.cpu().numpy()[0] + np.log(40)) < 1e-6
    for bad in (np.nan, np.inf):
        logits = np.zeros((2, 5000), np.float32)
        logits[1, 4321] = bad
        rt.logprobs_into(dev(logits), 2, 5000, t, f, None, 3, i, f)
        with pytest.raises(et.BackendError, match="logit 4321 of row 1 is NaN or"):
            rt.synchronize()
    rt.synchronize()
