"""Performance cases of a speculative decode step's operators, through the public Python entry
points: FP8 conversion and products with a scale for each block of 128, and the verification of
drafted tokens.

Kinds of call:
  quantize  Fp8Matrix.quantize and .dequantize: a matrix to 8-bit floating point (e4m3, with a
            power of two for each block) and back
  product   LmHeadFp8.logits: activations, quantised in the call, times a checkpoint's FP8 weights
  verify    DraftVerify: the drafted tokens that the target's distribution accepts, and one more

Each case is a dict of plain values; ``prepare`` makes its inputs on the GPU from a seed,
``run`` is one call (in plain torch operations while ``own`` is false), ``exact`` the same
outputs in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
LARGEST = 448.0  # of e4m3

# (temperature, top_k, top_p) of the requests, in turn; top_k 0: the whole vocabulary.
SAMPLING = {
    "pool": [(0.7, 40, 0.9)],
    "greedy": [(0.0, 1, 1.0)],
    "whole": [(1.0, 0, 1.0)],
    "nucleus": [(0.8, 0, 0.95)],
    "wide": [(1.0, 1000, 0.98)],
    "mixed": [(0.7, 40, 0.9), (1.0, 0, 1.0), (0.0, 1, 1.0), (0.8, 0, 0.95), (1.2, 100, 1.0), (1.0, 1000, 0.98)],
}


# ---------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------

def _quantize(rows, cols, dtype, block_rows):
    return {"kind": "quantize", "rows": rows, "cols": cols, "dtype": dtype, "block_rows": block_rows}


def _product(rows, n, k, dtype, out, bias=False):
    return {"kind": "product", "rows": rows, "n": n, "k": k, "dtype": dtype, "out": out, "bias": bias}


def _verify(requests, drafts, vocab, dtype, sampling, ragged=False, lookup=False):
    """`ragged`: the requests have from no drafted token to `drafts` of them. `lookup`: the drafts come without
    logits (looked up in the prompt)."""
    return {"kind": "verify", "requests": requests, "drafts": drafts, "vocab": vocab, "dtype": dtype,
            "sampling": sampling, "ragged": ragged, "lookup": lookup}


def _named(name, case):
    return {"name": name, **case}


def listed():
    return [
        # One token's hidden state to FP8 and back: latency.
        _named("quantize_token", _quantize(1, 896, "f32", 1)),
        # An odd batch of wide activations whose rows end inside a block.
        _named("quantize_ragged_bf16", _quantize(1531, 4850, "bf16", 1)),
        # A vocabulary's head converted when a model is loaded, in square blocks.
        _named("quantize_head_f16", _quantize(151936, 896, "f16", 128)),
        # The last layer of one sequence's decode step.
        _named("logits_one_token", _product(1, 151936, 896, "bf16", "f32")),
        # The target's logits for nine requests of four drafted tokens; sizes that fill no tile.
        _named("logits_drafts45", _product(45, 50257, 800, "f16", "f32", bias=True)),
        # A layer's projection for a short prompt.
        _named("project_prompt300", _product(300, 4864, 4096, "bf16", "bf16")),
        # A long prompt through a large layer: matrix work.
        _named("project_prompt4096", _product(4096, 16384, 4096, "bf16", "bf16")),
        # One chat request with four drafted tokens at the default sampling settings.
        _named("verify_one", _verify(1, 4, 151936, "f32", "pool")),
        # Tokens looked up in the prompt, from none to seven a request, drawn from the whole vocabulary.
        _named("verify_lookup_f16", _verify(17, 7, 50257, "f16", "whole", ragged=True, lookup=True)),
        # A batch of greedy requests.
        _named("verify_greedy_bf16", _verify(33, 5, 49152, "bf16", "greedy")),
        # Nucleus sampling over the whole vocabulary.
        _named("verify_nucleus", _verify(16, 4, 128000, "f32", "nucleus")),
        # A serving batch whose requests have settings of their own.
        _named("verify_batch", _verify(64, 4, 151936, "f32", "mixed", ragged=True)),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "verify", "verify", "verify"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "quantize":
        return _quantize(_between(rng, 1, 4096), _between(rng, 64, 8192), dtype, rng.choice([1, 128]))
    if kind == "product":
        rows, n, k = _between(rng, 1, 2048), _between(rng, 256, 65536), 8 * _between(rng, 32, 1024)
        n = min(n, max(256, 2 ** 37 // (rows * k)))
        return _product(rows, n, k, dtype, rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.4)
    drafts = rng.choice([1, 2, 3, 4, 5, 8])
    requests, vocab = _between(rng, 1, 256 // (drafts + 1)), _between(rng, 500, 151936)
    return _verify(requests, drafts, vocab, dtype, rng.choice(sorted(SAMPLING)), rng.random() < 0.5,
                   rng.random() < 0.3)


def _lengths(case):
    """The requests' numbers of drafted tokens."""
    if not case["ragged"]:
        return [case["drafts"]] * case["requests"]
    return [(5 * r + case["drafts"]) % (case["drafts"] + 1) for r in range(case["requests"])]


def _offsets(case):
    """Where the requests' rows of the target begin, and the last ones end."""
    at = [0]
    for n in _lengths(case):
        at.append(at[-1] + n + 1)
    return at


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _sampling_rows(case, counts):
    """temperature, top_k and top_p of each row, [rows, 1], for counts[r] rows of request r."""
    table = SAMPLING[case["sampling"]]
    rows = [table[r % len(table)] for r, n in enumerate(counts) for _ in range(n)]
    t, k, p = ([row[i] for row in rows] for i in range(3))
    k = [case["vocab"] if v == 0 else v for v in k]
    as_column = {"dtype": torch.float64, "device": "cuda"}
    return tuple(torch.tensor(v, **as_column).view(-1, 1) for v in (t, k, p))


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    kind = case["kind"]
    if kind == "quantize":
        # Activations or weights: normal, with a few channels much larger than the others.
        x = torch.randn(case["rows"], case["cols"], device="cuda", generator=g)
        x *= torch.exp(torch.randn(case["cols"], device="cuda", generator=g))
        state["x"] = x.to(DTYPES[case["dtype"]])
    elif kind == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        x = torch.randn(rows, k, device="cuda", generator=g)
        state["x"] = x.to(DTYPES[case["dtype"]])
        # A checkpoint's weights: e4m3 codes and a float32 scale, of any value, to each block.
        w = torch.randn(n, k, device="cuda", generator=g).mul_(100.0).clamp_(-LARGEST, LARGEST)
        codes = w.to(torch.float8_e4m3fn).view(torch.uint8)
        del w
        scales = torch.rand(-(-n // BLOCK), -(-k // BLOCK), device="cuda", generator=g)
        scales = (0.5 + scales) * (0.0002 / math.sqrt(k / 1024))
        state["bias"] = torch.randn(n, device="cuda", generator=g) if case["bias"] else None
        if own:
            from tabby_amd import fp8
            state["head"] = fp8.LmHeadFp8(fp8.Fp8Matrix.from_rowmajor(codes, scales), bias=state["bias"])
        else:
            state["codes"], state["scales"] = codes, scales
    else:
        requests, vocab, dtype = case["requests"], case["vocab"], DTYPES[case["dtype"]]
        lengths, at = _lengths(case), _offsets(case)
        rows, total = at[-1], at[-1] - requests
        x = torch.randn(rows, vocab, device="cuda", generator=g) * 2.0
        hot = torch.randint(0, vocab, (rows, 8), device="cuda", generator=g)
        x.scatter_(1, hot, 8.0 + 4.0 * torch.rand(rows, 8, device="cuda", generator=g))
        state["logits"] = x.to(dtype)
        # The target's row for each drafted token.
        before = torch.tensor([at[r] + j for r, n in enumerate(lengths) for j in range(n)], dtype=torch.int64,
                              device="cuda")
        state["draft_logits"] = None
        if total and not case["lookup"]:
            # A smaller model's logits: the target's, disturbed.
            y = x[before] + 0.6 * torch.randn(total, vocab, device="cuda", generator=g)
            state["draft_logits"] = y.to(dtype)
            del y
        del x
        # Drafted tokens are drawn from the draft's distribution; those looked up are often what the target says.
        source = state["draft_logits"] if state["draft_logits"] is not None else state["logits"][before]
        pick = torch.rand(total, 1, dtype=torch.float64, device="cuda", generator=g)
        drafts = torch.zeros(total, dtype=torch.int64, device="cuda")
        if total:
            drafts = _drawn(_distribution(source, *_sampling_rows(case, lengths)), pick)
        if case["lookup"]:
            other = torch.randint(0, vocab, (total,), device="cuda", generator=g)
            drafts = torch.where(torch.rand(total, device="cuda", generator=g) < 0.2, other, drafts)
        state["drafts"] = drafts.int()
        state["uniforms"] = torch.rand(total, dtype=torch.float64, device="cuda", generator=g)
        state["last"] = torch.rand(requests, dtype=torch.float64, device="cuda", generator=g)
        state["offsets"] = torch.tensor(at, dtype=torch.int32, device="cuda") if case["ragged"] else None
        if own:
            _prepare_verify(state, case)
    return state


def _prepare_verify(state, case):
    """The settings as the framework takes them, and the object with its workspace."""
    import numpy as np
    from tabby_amd import draft, sampler
    table = SAMPLING[case["sampling"]]
    settings = [sampler.SamplingParams(*table[r % len(table)]) for r in range(case["requests"])]
    params = sampler.make_params(settings, case["requests"], state["last"].cpu().numpy())
    state["params"] = torch.from_numpy(params.view(np.uint8).copy()).cuda()
    whole = any(s.temperature > 0 and (s.topK == 0 or s.topK > draft.POOL_MAX) for s in settings)
    state["flags"] = sampler.TABBY_FLAG_FULL_VOCAB if whole else 0
    state["verifier"] = draft.DraftVerify(vocab_max=case["vocab"], requests_max=case["requests"],
                                          drafts_max=case["drafts"])


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state, state["case"])
    return _PLAIN[kind](state, state["case"])


def _own_quantize(state, case):
    from tabby_amd import fp8
    m = fp8.Fp8Matrix.quantize(state["x"], block_rows=case["block_rows"])
    return m.dequantize(DTYPES[case["dtype"]])


def _own_product(state, case):
    return state["head"].logits(state["x"], dtype=DTYPES[case["out"]])


def _own_verify(state, case):
    v = state["verifier"](state["logits"], state["drafts"], state["params"], state["uniforms"],
                          draft_logits=state["draft_logits"], offsets=state["offsets"], flags=state["flags"])
    return v.tokens, v.accepted


def _round_blocks(x, block_rows):
    """The values, in 32 bits, that the matrix's blocks stand for once quantised."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK, 0, -rows % block_rows))
    v = v.view(-(-rows // block_rows), block_rows, -1, BLOCK)
    amax = v.abs().amax((1, 3), keepdim=True)
    # The smallest power of two with amax <= 448 times it; 448 is 7/8 of 2^9, and frexp's mantissa lies in [1/2, 1).
    mantissa, exponent = torch.frexp(amax)
    power = exponent - 9 + (mantissa > 0.875).int()
    power = torch.where(amax > 0, power.clamp_min(-126), torch.zeros_like(power))
    one = torch.ones_like(amax)
    a = v.abs() * torch.ldexp(one, -power)
    # A step is 2^-3 of the value's power of two, and 2^-9 below 2^-6.
    step = torch.ldexp(torch.ones_like(a), (torch.frexp(a).exponent - 1).clamp_min(-6) - 3)
    out = torch.copysign(torch.round(a / step) * step * torch.ldexp(one, power), v)
    out = torch.where(torch.isfinite(amax), out, torch.full_like(out, math.nan))
    return out.view(-1, out.shape[2] * BLOCK)[:rows, :cols]


def _plain_quantize(state, case):
    return _round_blocks(state["x"], case["block_rows"]).to(DTYPES[case["dtype"]])


def _plain_product(state, case):
    n, k = case["n"], case["k"]
    w = state["codes"].view(torch.float8_e4m3fn).float()
    w = w * state["scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = _round_blocks(state["x"], 1) @ w.t()
    if state["bias"] is not None:
        y = y + state["bias"]
    return y.to(DTYPES[case["out"]])


def _distribution(logits, temperature, top_k, top_p):
    """The probabilities that the sampler draws each row's token from, in 64 bits: whether a token is accepted,
    and which one is drawn, hangs on comparisons of sums."""
    x, ids = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    place = torch.arange(x.shape[1], device=x.device)
    greedy = temperature <= 0
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, temperature))
    w = torch.where(place < torch.where(greedy, 1.0, top_k), w, 0.0)
    reached = torch.cumsum(w, 1)
    before = reached - w
    kept = (before < top_p * reached[:, -1:]) | (top_p >= 1.0) | (place == 0)
    w = torch.where(kept, w, 0.0)
    return torch.zeros_like(w).scatter_(1, ids, w / w.sum(1, keepdim=True))


def _drawn(weights, uniform):
    """The first token, in the vocabulary's order, whose running sum exceeds its row's share of the total."""
    reached = torch.cumsum(weights, 1)
    above = reached > uniform * reached[:, -1:]
    last = (weights > 0).double().cumsum(1).argmax(1)
    return torch.where(above.any(1), above.int().argmax(1), last)


def _plain_verify(state, case):
    requests, drafts = case["requests"], case["drafts"]
    lengths, at = _lengths(case), _offsets(case)
    device = state["logits"].device
    p = _distribution(state["logits"], *_sampling_rows(case, [n + 1 for n in lengths]))
    length = torch.tensor(lengths, device=device)
    first = torch.tensor(at[:-1], device=device)
    first_draft = first - torch.arange(requests, device=device)
    tokens = state["drafts"].long()
    q = None
    if tokens.numel():
        owner = torch.repeat_interleave(torch.arange(requests, device=device), length)
        row = torch.arange(tokens.numel(), device=device) + owner
        share = p[row].gather(1, tokens[:, None])[:, 0]
        claimed = torch.ones_like(share)
        if state["draft_logits"] is not None:
            q = _distribution(state["draft_logits"], *_sampling_rows(case, lengths))
            claimed = q.gather(1, tokens[:, None])[:, 0]
        good = state["uniforms"] * claimed < share
    else:
        good = torch.zeros(0, dtype=torch.bool, device=device)
    # Drafts by request, those past the last one refused.
    place = torch.arange(drafts, device=device)
    inside = place[None] < length[:, None]
    index = (first_draft[:, None] + place[None]).clamp(0, max(tokens.numel() - 1, 0))
    pad = torch.zeros(1, dtype=torch.bool, device=device)
    run_ = inside & (good if tokens.numel() else pad)[index]
    accepted = run_.int().cumprod(1).sum(1)
    weights = p[first + accepted]
    refused = accepted < length
    if tokens.numel():
        at_draft = (first_draft + accepted).clamp_max(tokens.numel() - 1)
        if q is not None:
            taken = q[at_draft]
        else:
            taken = torch.zeros_like(weights).scatter_(1, tokens[at_draft][:, None], 1.0)
        rest = (weights - taken).clamp_min(0.0)
        rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, weights)
        weights = torch.where(refused[:, None], rest, weights)
    last = _drawn(weights, state["last"][:, None])
    out = torch.full((requests, drafts + 1), -1, dtype=torch.int64, device=device)
    kept = place[None] < accepted[:, None]
    if tokens.numel():
        out[:, :drafts] = torch.where(kept, tokens[index], -1)
    out.scatter_(1, accepted[:, None].long(), last[:, None])
    return out.int(), accepted.int()


_OWN = {"quantize": _own_quantize, "product": _own_product, "verify": _own_verify}
_PLAIN = {"quantize": _plain_quantize, "product": _plain_product, "verify": _plain_verify}


# ---------------------------------------------------------------------------------------
# What a pass cannot do without, and its outputs in 64 bits
# ---------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "quantize":
        rows, cols = case["rows"], case["cols"]
        held = rows * cols + 4 * -(-rows // case["block_rows"]) * -(-cols // BLOCK)
        return {"bytes": 2 * rows * cols * SIZES[case["dtype"]] + 2 * held, "flops": 4.0 * rows * cols}
    if kind == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        held = n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK)
        moved = rows * k * SIZES[case["dtype"]] + rows * n * SIZES[case["out"]] + (4 * n if case["bias"] else 0)
        return {"bytes": held + moved, "flops": 2.0 * rows * n * k}
    requests, rows = case["requests"], _offsets(case)[-1]
    total = rows - requests
    # Of the draft's logits, those of the requests that do not only take the largest.
    table = SAMPLING[case["sampling"]]
    drawn = sum(n for r, n in enumerate(_lengths(case)) if table[r % len(table)][0] > 0)
    read = (rows + (0 if case["lookup"] else drawn)) * case["vocab"] * SIZES[case["dtype"]]
    moved = 12 * total + 32 * requests + 4 * requests * (case["drafts"] + 2)
    return {"bytes": read + moved, "flops": 4.0 * read / SIZES[case["dtype"]]}


def _values_of_codes():
    """The 127 magnitudes of e4m3, in 64 bits."""
    out = [m / 8 * 2.0 ** -6 for m in range(8)]
    for e in range(1, 16):
        out += [(1 + m / 8) * 2.0 ** (e - 7) for m in range(8)]
    return out[:127]  # the last one is NaN


def _nearest(x, block_rows):
    """Values in 64 bits of the quantised matrix: the code by comparisons with the midpoints, half way to the even one."""
    levels = torch.tensor(_values_of_codes(), dtype=torch.float64, device=x.device)
    middles = (levels[:-1] + levels[1:]) / 2
    powers = torch.tensor([2.0 ** e for e in range(-126, 128)], dtype=torch.float64, device=x.device)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[1], BLOCK):
        v = x[:, c:c + BLOCK].double()
        largest = v.abs().amax(1)
        if block_rows > 1:
            groups = torch.arange(v.shape[0], device=x.device) // block_rows
            top = torch.zeros(int(groups[-1]) + 1, dtype=torch.float64, device=x.device)
            largest = top.scatter_reduce(0, groups, largest, "amax")[groups]
        power = powers[torch.searchsorted(powers, largest / LARGEST).clamp(0, 253)][:, None]
        a = v.abs() / power
        low = torch.searchsorted(middles, a)                 # an exact midpoint: the lower one
        high = torch.searchsorted(middles, a, right=True)    # and the upper one
        code = torch.where(low % 2 == 0, low, high)
        out[:, c:c + BLOCK] = torch.where(torch.isfinite(largest)[:, None], torch.copysign(levels[code] * power, v), math.nan)
    return out


def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    kind = case["kind"]
    if kind == "quantize":
        return _nearest(state["x"], case["block_rows"])
    if kind == "product":
        n, k, codes = case["n"], case["k"], state["codes"]
        levels = torch.tensor(_values_of_codes() + [math.nan], dtype=torch.float64, device="cuda")
        w = torch.empty(n, k, dtype=torch.float64, device="cuda")
        for c in range(0, k, BLOCK):
            part = codes[:, c:c + BLOCK].int()
            scale = state["scales"][torch.arange(n, device="cuda") // BLOCK, c // BLOCK].double()
            w[:, c:c + BLOCK] = levels[part & 127] * (1 - 2 * (part >> 7)) * scale[:, None]
        y = torch.mm(_nearest(state["x"], 1), w.t().contiguous())
        return y if state["bias"] is None else y + state["bias"].double()
    return _decided(state, case)


def _shares(row, setting):
    """(tokens, weights) that a row's token is drawn from, best first, not divided by their sum."""
    temperature, top_k, top_p = setting
    order = torch.argsort(row, descending=True, stable=True)
    if temperature <= 0:
        return order[:1], torch.ones(1, dtype=torch.float64, device=row.device)
    if top_k:
        order = order[:top_k]
    weights = torch.exp((row[order] - row[order[0]]) / temperature)
    if top_p < 1:
        sums = weights.cumsum(0)
        count = int((sums < top_p * sums[-1]).sum()) + 1
        order, weights = order[:count], weights[:count]
    return order, weights


def _decided(state, case):
    """Each request by itself, one drafted token after another."""
    at, table = _offsets(case), SAMPLING[case["sampling"]]
    tokens = torch.full((case["requests"], case["drafts"] + 1), -1, dtype=torch.int32)
    accepted = torch.zeros(case["requests"], dtype=torch.int32)
    drafts, uniforms, last = (state[name].tolist() for name in ("drafts", "uniforms", "last"))
    for r, length in enumerate(_lengths(case)):
        setting, begin = table[r % len(table)], at[r] - r
        rest = torch.zeros(case["vocab"], dtype=torch.float64, device="cuda")
        taken = 0
        while True:
            ids, weights = _shares(state["logits"][at[r] + taken].double(), setting)
            rest.zero_()
            rest[ids] = weights / weights.sum()
            if taken == length:
                break
            token = drafts[begin + taken]
            claim = torch.zeros_like(rest)
            if state["draft_logits"] is None:
                claim[token] = 1.0
            else:
                ids, weights = _shares(state["draft_logits"][begin + taken].double(), setting)
                claim[ids] = weights / weights.sum()
            if uniforms[begin + taken] * float(claim[token]) < float(rest[token]):
                tokens[r, taken] = token
                taken += 1
                continue
            left = torch.relu(rest - claim)
            if float(left.sum()) > 0:
                rest = left
            break
        sums = rest.cumsum(0)
        tokens[r, taken] = int(torch.searchsorted(sums, last[r] * float(sums[-1]), right=True))
        accepted[r] = taken
    return tokens.cuda(), accepted.cuda()
