"""Operators of long-context serving, as measurable cases: rotary positions scaled beyond the trained context, a paged KV cache
held in 4 bits (append, read back, attention), and log probabilities of given tokens.

own                 False: plain torch forms. True: the calls that a program makes of this library
listed()            the named cases
draw(rng)           one more case of the same ranges
prepare(case, seed) inputs, pages and handles a program holds before the call, made from the seed
run(state)          one pass; returns what the operator computes
work(case)          bytes and operations one pass cannot do without
exact(case, seed)   the outputs in 64 bits, from the operators' definitions

A 4-bit row is cut into blocks of 32 values. A block's scale is its value of largest magnitude (the first of equals) divided by -8, stored as
f16; a code is floor(x / scale + 8.5) held to 0..15, computed in f32 with the unrounded scale, and stands for (code - 8) * scale.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
VOCAB = 128256


def listed():
    return [
        # One decode step of 32 sequences far into an extended context: the query and key heads inside the fused projection's rows.
        dict(name="rope-step-b32", kind="rope", batch=32, steps=1, q_heads=32, kv_heads=8, head_dim=128, rotary=128, layout="half", scaling="llama3",
             theta=500000.0, factor=8.0, original=8192, reach=131072),
        # A prompt of 4096 tokens, 64 query heads, interleaved pairs, a window extended 32 times.
        dict(name="rope-prompt-4096", kind="rope", batch=1, steps=4096, q_heads=64, kv_heads=8, head_dim=128, rotary=128, layout="pairs", scaling="yarn",
             theta=10000.0, factor=32.0, original=4096, reach=65536),
        # Three ragged prompts of a small model that rotates three quarters of a head.
        dict(name="rope-part-b3", kind="rope", batch=3, steps=333, q_heads=4, kv_heads=2, head_dim=64, rotary=48, layout="half", scaling="linear",
             theta=10000.0, factor=4.0, original=2048, reach=8192),
        # The new rows of one decode step of 64 sequences go to their pages; then they are read back.
        dict(name="append-step-b64", kind="append", batch=64, tokens=1, kv_heads=8, head_dim=128, context=4096),
        # A chunk of every prompt of a batch, an odd number of tokens that starts and ends inside pages.
        dict(name="append-chunk-b8", kind="append", batch=8, tokens=509, kv_heads=8, head_dim=128, context=512),
        # The smallest call: the start of one conversation with a small model.
        dict(name="attention-37", kind="attention", batch=1, q_heads=4, kv_heads=2, head_dim=64, shortest=37, longest=37),
        # The batched decode shape: 64 sequences of 128 to 4096 tokens over shuffled pages.
        dict(name="attention-b64", kind="attention", batch=64, q_heads=32, kv_heads=8, head_dim=128, shortest=128, longest=4096),
        # One user with a context of 131072 tokens.
        dict(name="attention-131072", kind="attention", batch=1, q_heads=32, kv_heads=8, head_dim=128, shortest=131072, longest=131072),
        # The larger shape, 64 query heads, 16 long sequences.
        dict(name="attention-64h-b16", kind="attention", batch=16, q_heads=64, kv_heads=8, head_dim=128, shortest=1024, longest=16384),
        # One token with its alternatives, as a chat server returns them.
        dict(name="logprobs-1-top20", kind="logprobs", rows=1, vocab=VOCAB, top=20, masked=False),
        # A decode step of 32 sequences under a grammar that bars half of the vocabulary.
        dict(name="logprobs-32-top5", kind="logprobs", rows=32, vocab=VOCAB, top=5, masked=True),
        # Scoring a text: every position of a chunk, no alternatives.
        dict(name="logprobs-2048", kind="logprobs", rows=2048, vocab=VOCAB, top=0, masked=False),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("rope", "append", "attention", "attention", "logprobs"))
    head_dim = rng.choice((64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    q_heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 7, 8, 16) if kind == "attention" else (1, 2, 4, 8))
    if kind == "rope":
        batch = _spread(rng, 1, 64)
        steps = _spread(rng, 1, max(1, 4096 // batch))
        scaling = rng.choice(("none", "linear", "llama3", "yarn"))
        return dict(kind=kind, batch=batch, steps=steps, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                    rotary=rng.choice((head_dim, head_dim, head_dim // 2, head_dim // 4 * 3, 2 * rng.randint(1, head_dim // 2))),
                    layout=rng.choice(("half", "pairs")), scaling=scaling, theta=rng.choice((10000.0, 500000.0)), factor=rng.choice((2.0, 4.0, 8.0, 32.0)),
                    original=rng.choice((2048, 4096, 8192)), reach=_spread(rng, 4096, 1 << 20))
    if kind == "append":
        batch = _spread(rng, 1, 64)
        return dict(kind=kind, batch=batch, tokens=_spread(rng, 1, max(1, 4096 // batch)), kv_heads=kv_heads, head_dim=head_dim, context=_spread(rng, 1, 1024))
    if kind == "attention":
        batch = _spread(rng, 1, 64)
        longest = _spread(rng, 1, min(131072, 262144 // batch * 8 // kv_heads))
        return dict(kind=kind, batch=batch, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, shortest=max(1, int(longest * rng.choice((0.03, 0.5, 1.0)))),
                    longest=longest)
    vocab = rng.choice((VOCAB, 4096, 2048, _spread(rng, 33, 200000)))
    return dict(kind=kind, rows=_spread(rng, 1, min(2048, 2048 * VOCAB // vocab)), vocab=vocab, top=rng.choice((0, 0, 1, 5, 20, 32)), masked=rng.random() < 0.5)


def work(case):
    c = case
    if c["kind"] == "rope":  # heads in, heads out, a frequency per pair
        values = c["batch"] * c["steps"] * (c["q_heads"] + c["kv_heads"]) * c["head_dim"]
        return {"bytes": 8.0 * values + 8.0 * c["batch"], "flops": 3.0 * values}
    if c["kind"] == "append":  # K and V in; codes and scales out, and in again; values out
        values = 2 * c["batch"] * c["tokens"] * c["kv_heads"] * c["head_dim"]
        return {"bytes": values * (4 + 2 * 18 / 32 + 4), "flops": 4.0 * values}
    if c["kind"] == "attention":
        tokens = sum(_lengths(c))
        row = c["kv_heads"] * c["head_dim"] * 18 / 32
        return {"bytes": 2 * tokens * row + 8.0 * c["batch"] * c["q_heads"] * c["head_dim"], "flops": 4.0 * tokens * c["q_heads"] * c["head_dim"]}
    return {"bytes": 4.0 * c["rows"] * (c["vocab"] + 3 + 2 * c["top"]), "flops": 4.0 * c["rows"] * c["vocab"]}


def _lengths(case):
    """Cached tokens of each sequence: the first has the longest context, the others are even between the bounds."""
    n, low, high = case["batch"], case["shortest"], case["longest"]
    return [high - (high - low) * i // max(n - 1, 1) for i in range(n)]


# ---- inputs ---------------------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rows(case, lengths, seed):
    """K and V of each sequence in turn, f32 [kv_heads, length, head_dim]; keys of some columns are larger than of others, as after training."""
    g = _generator(seed + 1)
    column = torch.randn(2, case["kv_heads"], 1, case["head_dim"], generator=g, device="cuda").mul_(0.7).exp_()
    for n in lengths:
        both = torch.randn(2, case["kv_heads"], n, case["head_dim"], generator=g, device="cuda")
        yield both[0] * column[0], both[1] * column[1].mean()


def _tables(lengths, seed):
    """Pages of each sequence, from a shuffled pool: (numbers one sequence after the other, where each starts, pages in the pool)."""
    counts = [(n + PAGE - 1) // PAGE for n in lengths]
    total = sum(counts)
    pages = np.random.default_rng(seed + 2).permutation(total)
    return torch.from_numpy(pages.astype(np.int32)).cuda(), [sum(counts[:i]) for i in range(len(counts))], total


_runtime = None


def _the_runtime():
    global _runtime
    if _runtime is None:
        import effect_torch_b200 as et
        _runtime = et.Runtime(0)
    return _runtime


def _pool(case, pages):
    import effect_torch_b200 as et
    return et.NativeKvPool(_the_runtime(), 1, case["kv_heads"], case["head_dim"], pages * PAGE, PAGE, et.KV_Q4)


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case["kind"] == "rope":
        b, t, heads, d = case["batch"], case["steps"], case["q_heads"] + 2 * case["kv_heads"], case["head_dim"]
        s["qkv"] = torch.randn(b, t, heads, d, generator=g, device="cuda")
        s["offsets"] = torch.randint(0, max(1, case["reach"] - t), (b,), generator=g, device="cuda")
        if own:
            import effect_torch_b200 as et
            s["rope"] = et.RotaryTable(_the_runtime(), head_dim=d, rotary_dim=case["rotary"], theta=case["theta"],
                                       layout=et.HALF_SPLIT if case["layout"] == "half" else et.INTERLEAVED_PAIRS, scaling=case["scaling"], factor=case["factor"],
                                       original_context=case["original"])
            s["out"] = torch.empty(b, t, heads - case["kv_heads"], d, device="cuda")
        else:
            s["frequencies"], s["magnitude"] = _frequencies(case)
        return s
    if case["kind"] == "append":
        b, t, h, d = case["batch"], case["tokens"], case["kv_heads"], case["head_dim"]
        before = [case["context"] * (i + 1) // b for i in range(b)]
        s["k"], s["v"] = (torch.randn(b, h, t, d, generator=g, device="cuda") for _ in range(2))
        if own:
            table, first, pages = _tables([n + t for n in before], seed)
            s["pool"], s["tables"] = _pool(case, pages), table
            s["lanes"] = torch.tensor([[n, t, 0, f] for n, f in zip(before, first)], dtype=torch.int32, device="cuda")
            at = torch.tensor(before, device="cuda")[:, None] + torch.arange(t, device="cuda")
            page = table[torch.tensor(first, device="cuda")[:, None] + at // PAGE].long()
            s["rows"] = (page * PAGE + at % PAGE).reshape(-1).int()
            s["out"] = torch.empty(2, b * t, h * d, device="cuda")
        return s
    if case["kind"] == "attention":
        lengths = _lengths(case)
        h, d = case["kv_heads"], case["head_dim"]
        s["q"] = torch.randn(case["batch"], case["q_heads"], d, generator=g, device="cuda")
        if own:
            rt = _the_runtime()
            table, first, pages = _tables(lengths, seed)
            s["pool"], s["tables"] = _pool(case, pages), table
            for n, at, (k, v) in zip(lengths, first, _rows(case, lengths, seed)):
                lane = torch.tensor([[0, n, 0, at]], dtype=torch.int32, device="cuda")
                torch.cuda.synchronize()
                rt.paged_append_into(s["pool"], 0, lane, table, 1, n, k, v)
                rt.synchronize()
            s["lanes"] = torch.tensor([[n - 1, 1, 0, f] for n, f in zip(lengths, first)], dtype=torch.int32, device="cuda")
            s["pages"] = (lengths[0] + PAGE - 1) // PAGE
            s["scratch_bytes"] = s["pool"].attention_scratch_bytes(case["batch"], case["q_heads"], s["pages"])
            s["scratch"] = torch.empty(max(s["scratch_bytes"], 1), dtype=torch.uint8, device="cuda")
            s["out"] = torch.empty(case["batch"], case["q_heads"], d, device="cuda")
        else:
            n = lengths[0]
            s["codes"] = torch.zeros(2, case["batch"], h, n, d, dtype=torch.int8, device="cuda")
            s["scales"] = torch.zeros(2, case["batch"], h, n, d // 32, dtype=torch.float16, device="cuda")
            s["lengths"] = torch.tensor(lengths, device="cuda")
            for i, both in enumerate(_rows(case, lengths, seed)):
                for side, x in enumerate(both):
                    s["codes"][side, i, :, :lengths[i]], s["scales"][side, i, :, :lengths[i]] = _quantize(x)
        return s
    rows, vocab = case["rows"], case["vocab"]
    # a head's logits; the alternatives of a row tie now and then, as those of a head with few bits do
    s["logits"] = torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.5)
    if rows * vocab <= 1 << 26:
        s["logits"] = s["logits"].mul_(64).round_().div_(64)
    s["targets"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    if case["masked"]:
        barred = torch.rand(rows, vocab, generator=g, device="cuda") < 0.5
        barred.scatter_(1, s["targets"].long()[:, None], False)
        s["logits"].masked_fill_(barred, -math.inf)
    if own:
        s["logprobs"], s["entropy"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        s["tokens"] = torch.empty(rows, min(case["top"], vocab), dtype=torch.int32, device="cuda")
        s["alternatives"] = torch.empty(rows, min(case["top"], vocab), device="cuda")
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _RUN[s["kind"]](s)
    return _PLAIN[s["kind"]](s)


def _run_rope(s):
    b, t, heads, d = s["qkv"].shape
    rotated = heads - s["kv_heads"]
    _the_runtime().rotary_into(s["rope"], s["qkv"], s["offsets"], b, rotated, t, s["out"], x_strides=(t * heads * d, d, heads * d),
                               out_strides=(t * rotated * d, d, rotated * d))
    return s["out"]


def _run_append(s):
    rt = _the_runtime()
    rt.paged_append_into(s["pool"], 0, s["lanes"], s["tables"], s["batch"], s["tokens"], s["k"], s["v"])
    for side in (0, 1):
        rt.pool_rows_into(s["pool"], 0, side, s["rows"], s["rows"].numel(), s["out"][side])
    return s["out"]


def _run_attention(s):
    _the_runtime().paged_attention_into(s["pool"], 0, s["lanes"], s["tables"], s["batch"], s["pages"], s["q"], s["q_heads"], s["head_dim"] ** -0.5, s["out"],
                                        s["scratch"], s["scratch_bytes"])
    return s["out"]


def _run_logprobs(s):
    _the_runtime().logprobs_into(s["logits"], s["rows"], s["vocab"], s["targets"], s["logprobs"], s["entropy"], s["tokens"].shape[1], s["tokens"], s["alternatives"])
    return {"logprobs": s["logprobs"], "entropy": s["entropy"], "tokens": s["tokens"], "alternatives": s["alternatives"]}


_RUN = {"rope": _run_rope, "append": _run_append, "attention": _run_attention, "logprobs": _run_logprobs}


def _frequencies(c):
    """Angle per position of each rotated pair, f64, and the factor on the rotated values."""
    pairs = c["rotary"] // 2
    f = c["theta"] ** (-2.0 * torch.arange(pairs, dtype=torch.float64, device="cuda") / c["rotary"])
    if c["scaling"] == "linear":
        return f / c["factor"], 1.0
    if c["scaling"] == "llama3":  # long wavelengths are stretched, short ones stay, those between go over from one to the other
        turns = c["original"] * f / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * ((1 - smooth) / c["factor"] + smooth), 1.0
    if c["scaling"] == "yarn":
        def corner(turns):
            return c["rotary"] * math.log(c["original"] / (turns * 2 * math.pi)) / (2 * math.log(c["theta"]))
        low, high = max(math.floor(corner(32.0)), 0), min(math.ceil(corner(1.0)), c["rotary"] - 1)
        ramp = ((torch.arange(pairs, dtype=torch.float64, device="cuda") - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / c["factor"] * ramp + f * (1 - ramp), 0.1 * math.log(c["factor"]) + 1.0
    return f, 1.0


def _plain_rope(s):
    x = s["qkv"][:, :, : s["q_heads"] + s["kv_heads"]]
    r = s["rotary"]
    position = s["offsets"][:, None] + torch.arange(s["steps"], device="cuda")
    angle = (position.double()[:, :, None] * s["frequencies"])[:, :, None]
    cosine, sine = ((f(angle) * s["magnitude"]).float() for f in (torch.cos, torch.sin))
    out = x.clone()
    a, b = (slice(0, r // 2), slice(r // 2, r)) if s["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
    out[..., a] = x[..., a] * cosine - x[..., b] * sine
    out[..., b] = x[..., b] * cosine + x[..., a] * sine
    return out


def _quantize(x):
    """Codes less 8 (int8), like x, and scales (f16) of its blocks of 32."""
    block = x.reshape(*x.shape[:-1], -1, 32)
    magnitude = block.abs()
    largest = magnitude == magnitude.amax(-1, keepdim=True)
    first = torch.where(largest, torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    scale = block.gather(-1, first) * -0.125
    inverse = torch.where(scale != 0, 1 / scale, torch.zeros_like(scale))
    code = (block * inverse).add_(8.5).floor_().clamp_(0, 15).sub_(8)
    return code.to(torch.int8).reshape(x.shape), scale.half()[..., 0]


def _values(codes, scales):
    return (codes.reshape(*scales.shape, 32).float() * scales.float()[..., None]).reshape(codes.shape)


def _plain_append(s):
    sides = (_values(*_quantize(x)).transpose(1, 2).reshape(s["batch"] * s["tokens"], -1) for x in (s["k"], s["v"]))
    return torch.stack(tuple(sides))


def _plain_attention(s):
    b, h, d = s["batch"], s["kv_heads"], s["head_dim"]
    k, v = (_values(s["codes"][side], s["scales"][side]) for side in (0, 1))
    scores = (s["q"] * d ** -0.5).reshape(b, h, -1, d) @ k.transpose(-1, -2)
    live = torch.arange(k.shape[2], device="cuda") < s["lengths"][:, None]
    scores = scores.masked_fill(~live[:, None, None], -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True)).exp()
    return ((weights @ v) / weights.sum(-1, keepdim=True)).reshape(b, -1, d)


def _plain_logprobs(s):
    x = s["logits"]
    largest = x.amax(-1, keepdim=True)
    shifted = x - largest
    weights = shifted.exp()
    total = weights.sum(-1, keepdim=True)
    entropy = total.log() - (weights * shifted.nan_to_num(neginf=0.0)).sum(-1, keepdim=True) / total
    base = largest + total.log()
    # of equal values the lower token comes first
    best, order = x.sort(dim=-1, descending=True, stable=True) if s["top"] else (x[:, :0], x[:, :0])
    top = min(s["top"], s["vocab"])
    return {"logprobs": (x.gather(-1, s["targets"].long()[:, None]) - base)[:, 0], "entropy": entropy[:, 0], "tokens": order[:, :top].int(),
            "alternatives": best[:, :top] - base}


_PLAIN = {"rope": _plain_rope, "append": _plain_append, "attention": _plain_attention, "logprobs": _plain_logprobs}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------

def exact(case, seed):
    g = _generator(seed)
    c = case
    if c["kind"] == "rope":
        b, t, d, r = c["batch"], c["steps"], c["head_dim"], c["rotary"]
        x = torch.randn(b, t, c["q_heads"] + 2 * c["kv_heads"], d, generator=g, device="cuda")[:, :, : c["q_heads"] + c["kv_heads"]].double()
        offsets = torch.randint(0, max(1, c["reach"] - t), (b,), generator=g, device="cuda")
        frequency, magnitude = [], 1.0
        for j in range(r // 2):
            f = 1.0 / math.pow(c["theta"], 2 * j / r)
            if c["scaling"] == "linear":
                f /= c["factor"]
            elif c["scaling"] == "llama3":
                wavelength = 2 * math.pi / f
                if wavelength > c["original"]:
                    f /= c["factor"]
                elif wavelength > c["original"] / 4:
                    part = (c["original"] / wavelength - 1) / 3
                    f = (1 - part) * f / c["factor"] + part * f
            elif c["scaling"] == "yarn":
                magnitude = 1.0 + math.log(c["factor"]) / 10
                edge = [r * math.log(c["original"] / (2 * math.pi * n)) / (2 * math.log(c["theta"])) for n in (32, 1)]
                low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), r - 1)
                kept = 1 - min(1.0, max(0.0, (j - low) / (high - low if high > low else 0.001)))
                f = f / c["factor"] * (1 - kept) + f * kept
            frequency.append(f)
        turn = torch.polar(torch.tensor(magnitude, dtype=torch.float64, device="cuda"),
                           (offsets[:, None] + torch.arange(t, device="cuda")).double()[..., None] * torch.tensor(frequency, dtype=torch.float64, device="cuda"))
        out = x.clone()
        if c["layout"] == "half":
            z = torch.complex(x[..., : r // 2], x[..., r // 2:r]) * turn[:, :, None]
            out[..., :r] = torch.cat((z.real, z.imag), -1)
        else:
            z = torch.view_as_complex(x[..., :r].reshape(b, t, -1, r // 2, 2)) * turn[:, :, None]
            out[..., :r] = torch.view_as_real(z).flatten(-2)
        return out
    if c["kind"] == "append":
        b, t = c["batch"], c["tokens"]
        sides = [torch.randn(b, c["kv_heads"], t, c["head_dim"], generator=g, device="cuda") for _ in range(2)]
        return torch.stack([_stored(x).transpose(1, 2).reshape(b * t, -1) for x in sides])
    if c["kind"] == "attention":
        lengths = _lengths(c)
        q = torch.randn(c["batch"], c["q_heads"], c["head_dim"], generator=g, device="cuda").double()
        out = torch.empty_like(q)
        for i, (k, v) in enumerate(_rows(c, lengths, seed)):
            for j in range(c["kv_heads"]):
                mine = slice(j * c["q_heads"] // c["kv_heads"], (j + 1) * c["q_heads"] // c["kv_heads"])
                keys, values = _stored(k[j]), _stored(v[j])
                out[i, mine] = torch.softmax(torch.einsum("gd,nd->gn", q[i, mine], keys) / math.sqrt(c["head_dim"]), -1) @ values
        return out
    logits = torch.randn(c["rows"], c["vocab"], generator=g, device="cuda").mul_(2.5)
    if c["rows"] * c["vocab"] <= 1 << 26:
        logits = logits.mul_(64).round_().div_(64)
    targets = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device="cuda", dtype=torch.int32).long()
    barred = torch.rand(c["rows"], c["vocab"], generator=g, device="cuda") < 0.5 if c["masked"] else None
    top = min(c["top"], c["vocab"])
    found = {"logprobs": [], "entropy": [], "alternatives": []}
    for i in range(c["rows"]):
        row = logits[i].double()
        if barred is not None:
            row[barred[i] & (torch.arange(c["vocab"], device="cuda") != targets[i])] = -math.inf
        row = torch.log_softmax(row, -1)
        found["logprobs"].append(row[targets[i]])
        found["entropy"].append(-torch.xlogy(row.exp(), row.exp()).sum())
        found["alternatives"].append(row.topk(top).values)
    return {"logprobs": torch.stack(found["logprobs"]), "entropy": torch.stack(found["entropy"]), "tokens": None, "alternatives": torch.stack(found["alternatives"])}


def _stored(x):
    """The values that 4-bit rows of x stand for, f64. The choice of codes is defined in f32."""
    block = x.reshape(-1, 32)
    size = block.abs()
    # the first of the largest: the one whose mark weighs most
    first = ((size == size.max(1, keepdim=True).values) * torch.arange(32, 0, -1, device=x.device)).argmax(1)
    scale = block[torch.arange(len(block), device=x.device), first] / -8
    code = torch.floor(block * torch.where(scale == 0, scale, scale.reciprocal())[:, None] + 8.5)
    return ((code.clamp(0, 15) - 8).double() * scale.half().double()[:, None]).reshape(x.shape)
