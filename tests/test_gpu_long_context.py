"""Decoders with scaled positions, 4-bit caches and scoring: whole steps against a plain Llama-shaped model in 64 bits.

The plain model attends over the rows that the decoder's cache holds (read back), after checking that each is what its own key or value
row is kept as, give or take a step of its block: a row whose f32 or f16 rounding differs may take the neighbouring code, and both are right.
Logits are held to what the decoder is held to elsewhere: 1e-5 (reference-order f32) and 2e-3 (f16 activations) of the largest."""
import re

import numpy as np
import pytest

import effect_torch_b200 as et
import oracle as orc
from tests import helpers
from tests.gpu_util import runtime

pytestmark = pytest.mark.gpu
PAGE = 16
SMALL = dict(layers=2, d_model=256, q_heads=4, kv_heads=2, head_dim=64, ffn=688, vocab=1500, rms_eps=1e-5, rope_theta=10000.0)
SMALL_Q = dict(helpers.TINY_Q, layers=2)
WIDE_Q = dict(layers=1, d_model=512, q_heads=8, kv_heads=1, head_dim=128, ffn=512, vocab=777, rms_eps=1e-5, rope_theta=500000.0)
RULES = {"plain": None, "half-part": dict(rotary_dim=32, layout=et.HALF_SPLIT), "pairs-part": dict(rotary_dim=46, layout=et.INTERLEAVED_PAIRS),
         "llama3": dict(scaling="llama3", factor=8.0, original_context=64), "yarn": dict(scaling="yarn", factor=4.0, original_context=200, layout=et.INTERLEAVED_PAIRS),
         "linear": dict(scaling="linear", factor=4.0, attention_factor=1.3)}


def dense(entry, codec):
    if isinstance(entry, tuple):
        return orc.dequantize(codec, *entry[:3]).astype(np.float64)
    return entry.astype(np.float64)


def rotate(x, position, config, divisors):
    """x [heads, rows, D] at positions [rows]."""
    f, m = et.rope_frequencies(config, divisors)
    r = config.rotary_dim
    angle = position[:, None] * f
    a, b = (slice(0, r // 2), slice(r // 2, r)) if config.layout == et.HALF_SPLIT else (slice(0, r, 2), slice(1, r, 2))
    out = x.copy()
    out[..., a] = m * (x[..., a] * np.cos(angle) - x[..., b] * np.sin(angle))
    out[..., b] = m * (x[..., b] * np.cos(angle) + x[..., a] * np.sin(angle))
    return out


class Plain:
    def __init__(self, cfg, weights, config, divisors, window=None):
        self.cfg, self.config, self.divisors, self.window = cfg, config, divisors, window
        codec = weights["codec"]
        self.w = {"tok_embd": weights["tok_embd"].astype(np.float64), "head": dense(weights["head"], codec),
                  "layers": [{k: dense(v, codec) for k, v in layer.items()} for layer in weights["layers"]]}

    def norm(self, x):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.cfg["rms_eps"])

    def logits(self, pool, seq, tokens, before, tier, room):
        """Logits of every token of a step that began at position `before` and whose rows are in the pool."""
        c = self.cfg
        D, Hq, Hkv = c["head_dim"], c["q_heads"], c["kv_heads"]
        n = len(tokens)
        position = before + np.arange(n)
        blocks, _ = seq.blocks
        rows = blocks[np.arange(before + n) // PAGE] * PAGE + np.arange(before + n) % PAGE
        x = self.w["tok_embd"][tokens]
        for l, w in enumerate(self.w["layers"]):
            h = self.norm(x)
            heads = lambda m, k: (h @ m.T).reshape(n, k, D).transpose(1, 0, 2)
            q, k, v = rotate(heads(w["wq"], Hq), position, self.config, self.divisors), rotate(heads(w["wk"], Hkv), position, self.config, self.divisors), heads(w["wv"], Hkv)
            cached = [pool.read_rows(l, which, rows).reshape(before + n, Hkv, D).transpose(1, 0, 2).astype(np.float64) for which in (0, 1)]
            for mine, kept in ((k, cached[0]), (v, cached[1])):
                off = np.abs(kept[:, before:] - mine)
                if tier == et.KV_Q4:  # half a step, a whole one at the far end of the range; what rounding moves on top
                    step = np.abs(mine).reshape(Hkv, n, D // 32, 32).max(-1, keepdims=True) / 8
                    assert (off.reshape(Hkv, n, D // 32, 32) <= 1.02 * step + room * np.abs(mine).max()).all()
                else:
                    assert off.max() <= ({et.KV_F32: 0, et.KV_F16: 2 ** -11, et.KV_BF16: 2 ** -8, et.KV_U8: 1 / 127}[tier] + room) * np.abs(mine).max()
            out = np.empty((n, Hq, D))
            for i in range(n):
                # the window's start for a whole step is that of its last token: what lies before is no longer resident
                begin = max(0, before + n - self.window) if self.window else 0
                for head in range(Hq):
                    kk, vv = (s[head // (Hq // Hkv), begin:before + i + 1] for s in cached)
                    s = kk @ q[head, i] / np.sqrt(D)
                    p = np.exp(s - s.max())
                    out[i, head] = p @ vv / p.sum()
            x = x + out.reshape(n, -1) @ w["wo"].T
            h = self.norm(x)
            gate, up = h @ w["gate"].T, h @ w["up"].T
            x = x + (gate / (1 + np.exp(-gate)) * up) @ w["down"].T
        return self.norm(x) @ self.w["head"].T


def make(cfg, weights, batch, tier, exact, rule, divisors=None, max_tokens=512, max_advance=64, window=None):
    config = et.rope_config(cfg["head_dim"], theta=cfg["rope_theta"]) if rule is None else et.rope_config(cfg["head_dim"], theta=cfg["rope_theta"], **rule)
    dec = et.Executable(runtime(), **cfg, batch=batch, max_tokens=max_tokens, block_size=PAGE, kv_dtype=tier, exact=exact, max_advance=max_advance, window=window,
                        rope=None if rule is None else config, rope_divisors=divisors)
    helpers.load_into(dec, weights)
    dec.finalize()
    pool = et.NativeKvPool(runtime(), cfg["layers"], cfg["kv_heads"], cfg["head_dim"], max_tokens, PAGE, tier)
    return dec, pool, Plain(cfg, weights, config, divisors, window)


def run(dec, pool, plain, tier, tol, steps, batch, scored=False, seed=0, room=None):
    rng = np.random.default_rng(seed)
    seqs, vocab = [pool.makeSequence() for _ in range(batch)], plain.cfg["vocab"]
    before = 0
    for advance in steps:
        tokens = rng.integers(0, vocab, (batch, advance)).astype(np.uint32)
        if scored:
            targets = rng.integers(0, vocab, (batch, advance)).astype(np.uint32)
            lp, entropy, top_tokens, top_lp = dec.score(pool, seqs, tokens, targets, top=5)
        else:
            got = dec.execute(pool, seqs, tokens)
        assert [s.cursor for s in seqs] == [before + advance] * batch
        for i, seq in enumerate(seqs):
            want = plain.logits(pool, seq, tokens[i], before, tier, tol if room is None else room)
            slack = tol * np.abs(want).max()
            if not scored:
                assert np.abs(got[i] - want[-1]).max() <= slack, (advance, np.abs(got[i] - want[-1]).max() / np.abs(want).max())
                continue
            ref = want - want.max(1, keepdims=True)
            ref -= np.log(np.exp(ref).sum(1, keepdims=True))
            # a log probability moves by at most the largest change of a logit, twice: its own and the sum's
            np.testing.assert_allclose(lp[i], ref[np.arange(advance), targets[i]], rtol=0, atol=2 * slack + 2e-5)
            p = np.exp(ref)
            # dH = -sum p (lp + H) dx, so at most max |dx| sum p |lp + H|
            h = -(p * ref).sum(1)
            np.testing.assert_allclose(entropy[i], h, rtol=0, atol=2e-5 + 1.1 * slack * (p * np.abs(ref + h[:, None])).sum(1).max())
            np.testing.assert_allclose(top_lp[i], np.take_along_axis(ref, top_tokens[i].astype(np.int64), 1), rtol=0, atol=2 * slack + 2e-5)
            best = -np.sort(-ref, axis=1)[:, :5]
            np.testing.assert_allclose(top_lp[i], best, rtol=0, atol=2 * slack + 2e-5)
        before += advance
    return seqs


@pytest.mark.parametrize("tier", [et.KV_F32, et.KV_F16, et.KV_U8, et.KV_Q4])
@pytest.mark.parametrize("rule", RULES)
def test_positions_of_reference_order_steps(rule, tier):
    w = helpers.make_weights(SMALL, seed=1)
    dec, pool, plain = make(SMALL, w, 2, tier, True, RULES[rule])
    run(dec, pool, plain, tier, 1e-5, (7, 1, 1, 64, 3, 1), 2)


@pytest.mark.parametrize("tier", [et.KV_F16, et.KV_BF16, et.KV_U8, et.KV_Q4])
@pytest.mark.parametrize("rule", RULES)
def test_positions_of_tensor_core_steps(rule, tier):
    w = helpers.make_weights(SMALL_Q, seed=2, codec=orc.Q4_0)
    dec, pool, plain = make(SMALL_Q, w, 2, tier, False, RULES[rule])
    run(dec, pool, plain, tier, 2e-2 if tier == et.KV_BF16 else 2e-3, (7, 1, 1, 64, 3, 1, 1), 2)


@pytest.mark.parametrize("exact", [True, False])
def test_frequency_divisors(exact):
    cfg = SMALL if exact else SMALL_Q
    w = helpers.make_weights(cfg, seed=3, codec=0 if exact else orc.Q8_0)
    dec, pool, plain = make(cfg, w, 2, et.KV_F16, exact, dict(), divisors=np.linspace(1, 8, 32))
    run(dec, pool, plain, et.KV_F16, 1e-5 if exact else 2e-3, (9, 1, 5, 1), 2)


@pytest.mark.parametrize("cfg", [SMALL_Q, WIDE_Q])
def test_long_generation_over_a_4_bit_cache(cfg):
    """Prompts of several chunks and steps whose tables outgrow the plan for short ones; one-token steps replay a captured graph."""
    w = helpers.make_weights(cfg, seed=4, codec=orc.Q4_0)
    dec, pool, plain = make(cfg, w, 2, et.KV_Q4, False, RULES["llama3"], max_tokens=1024)
    run(dec, pool, plain, et.KV_Q4, 2e-3, (64, 64, 64, 50, 1, 1, 1, 64, 64, 1, 1), 2)
    dec2, pool2, plain2 = make(cfg, w, 2, et.KV_Q4, False, None, max_tokens=512, window=100)
    run(dec2, pool2, plain2, et.KV_Q4, 2e-3, (64, 30, 1, 1, 20, 1, 1), 2)


def test_padded_lanes_and_device_resident_generation_over_a_4_bit_cache():
    cfg = SMALL_Q
    w = helpers.make_weights(cfg, seed=5, codec=orc.Q4_0)
    dec, pool, plain = make(cfg, w, 4, et.KV_Q4, False, RULES["yarn"])
    seqs = run(dec, pool, plain, et.KV_Q4, 2e-3, (40, 1, 1), 2)
    rng = np.random.default_rng(1)
    other = [pool.makeSequence() for _ in range(2)]
    prompt = rng.integers(0, cfg["vocab"], (2, 17)).astype(np.uint32)
    dec.execute(pool, other, prompt)
    a, b = (dec.executeSampled(pool, [s], [[5]]) for s in (seqs[0], other[0]))
    tokens, _ = dec.generate_greedy(pool, [seqs[0], other[0]], [a[0], b[0]], 12)
    # the same steps one by one, on sequences of their own
    again = [pool.makeSequence() for _ in range(2)]
    rng = np.random.default_rng(0)
    for advance in (40, 1, 1):
        t = rng.integers(0, cfg["vocab"], (2, advance)).astype(np.uint32)
        dec.execute(pool, [again[0]], t[:1])
    dec.execute(pool, [again[1]], prompt[:1])
    current = np.array([dec.executeSampled(pool, [s], [[5]])[0] for s in again])
    np.testing.assert_array_equal(current, [a[0], b[0]])
    for step in range(12):
        logits = dec.execute(pool, again, current[:, None])
        for i in range(2):  # equal, or a tie within what the plans' orders of sums differ by
            assert logits[i].max() - logits[i, tokens[step, i]] <= 4e-3 * np.abs(logits[i]).max()
        current = tokens[step]


@pytest.mark.parametrize("exact,tier", [(True, et.KV_F32), (False, et.KV_F16), (False, et.KV_Q4)])
def test_scores_of_a_text(exact, tier):
    cfg = SMALL if exact else SMALL_Q
    w = helpers.make_weights(cfg, seed=6, codec=0 if exact else orc.Q4_0)
    dec, pool, plain = make(cfg, w, 3, tier, exact, RULES["linear"])
    run(dec, pool, plain, tier, 1e-5 if exact else 2e-3, (5, 1, 64, 1, 2), 3, scored=True)
    seqs = run(dec, pool, plain, tier, 1e-5 if exact else 2e-3, (11, 1), 1, scored=True, seed=9)  # fewer sequences than lanes
    # scoring and executing are the same step
    tokens = np.array([[3, 1, 4]], np.uint32)
    twin = [pool.makeSequence()]
    rng = np.random.default_rng(9)
    for advance in (11, 1):
        dec.execute(pool, twin, rng.integers(0, cfg["vocab"], (1, advance)).astype(np.uint32))
        rng.integers(0, cfg["vocab"], (1, advance))
    lp = dec.score(pool, seqs, tokens, [[1, 4, 1]])[0]
    logits = dec.execute(pool, twin, tokens)[0].astype(np.float64)
    ref = logits[1] - logits.max() - np.log(np.exp(logits - logits.max()).sum())
    assert abs(lp[0, 2] - ref) <= (1e-5 if exact else 4e-3) * np.abs(logits).max() + 2e-5


def test_more_rows_than_logits_exist_at_a_time():
    cfg = dict(SMALL_Q, layers=1)
    w = helpers.make_weights(cfg, seed=7, codec=orc.Q4_0)
    dec, pool, plain = make(cfg, w, 5, et.KV_F16, False, None, max_tokens=640, max_advance=64)
    run(dec, pool, plain, et.KV_F16, 2e-3, (64, 64), 5, scored=True)  # 320 rows: 256 and 64


def test_a_bad_logit_is_reported_with_its_row():
    """Row of the step (lane 4's are 256 to 319), not of the 256 rows whose logits exist at a time. In f32: activations in f16 are held to
    finite numbers, so that a NaN does not reach their logits."""
    cfg = dict(SMALL, layers=1)
    w = helpers.make_weights(cfg, seed=7)
    w["tok_embd"][77] = np.nan
    dec, pool, _ = make(cfg, w, 5, et.KV_F32, True, None, max_tokens=640, max_advance=64)
    tokens = np.random.default_rng(1).integers(0, 77, (5, 64)).astype(np.uint32)
    tokens[4, 60] = 77
    seqs = [pool.makeSequence() for _ in range(5)]
    with pytest.raises(et.BackendError, match="logit") as e:
        dec.score(pool, seqs, tokens, tokens)
    assert 256 <= int(re.search(r"of row (\d+) is NaN", str(e.value)).group(1)) < 320
    assert [s.cursor for s in seqs] == [0] * 5


def test_a_step_that_fails_changes_nothing():
    cfg = SMALL
    w = helpers.make_weights(cfg, seed=8)
    dec, pool, plain = make(cfg, w, 2, et.KV_Q4, True, None, max_tokens=64)
    seqs = [pool.makeSequence()]
    good = np.array([[1, 2, 3]], np.uint32)
    for targets, top, cancelled, message in (([[1, 2, 1500]], 0, False, r"target 1500 is outside 0\.\.1500"), ([[1, 2, 3]], 33, False, "alternatives must be in"),
                                             ([[1, 2, 3]], -1, False, "alternatives must be in"), ([[1, 2, 3]], 0, True, "operation aborted"), ([[1, 2]], 0, False, "targets of shape")):
        with pytest.raises(et.BackendError, match=message):
            dec.score(pool, seqs, good, targets, top=top, cancelled=cancelled)
        assert seqs[0].cursor == 0 and seqs[0].frontier == 0
    with pytest.raises(et.BackendError, match="chunk of 65 tokens"):
        dec.score(pool, seqs, np.zeros((1, 65)), np.zeros((1, 65)))
    with pytest.raises(et.BackendError, match="accepts 1..=2"):
        dec.score(pool, [pool.makeSequence() for _ in range(3)], np.zeros((3, 1)), np.zeros((3, 1)))
    with pytest.raises(et.BackendError, match="1500 is outside"):
        dec.score(pool, seqs, [[1500]], [[0]])  # an embedding index
    assert seqs[0].cursor == 0
    dec.score(pool, seqs, good, [[1, 2, 3]])
    with pytest.raises(et.BackendError, match="must be null|are fixed"):
        et._check(runtime().L.etc_decoder_set_rope(dec.h, et.C.byref(et.rope_config(64)), None))
    for rope, message in ((et.rope_config(128), "head dimension of 128"), (et.rope_config(64, rotary_dim=65), "rotated part")):
        with pytest.raises(et.BackendError, match=message):
            et.Executable(runtime(), **SMALL, batch=1, max_tokens=64, rope=rope)
    with pytest.raises(et.BackendError, match="multiple of 32"):
        et.Executable(runtime(), **dict(SMALL, head_dim=40, d_model=160), batch=1, max_tokens=64, kv_dtype=et.KV_Q4)
