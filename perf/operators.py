"""Performance cases of the decode step's beam-search and MXFP4 operators, through the public
Python entry points.

Kinds of call:
  quantize  Mx4Matrix.quantize and .dequantize: a matrix to microscaled 4-bit floating point
            (blocks of 32 values with a shared power of two) and back
  product   LmHeadMx4.logits: activations, quantised in the call, times MXFP4 weights
  select    BeamSelect: the best continuations over the beams and the vocabulary of each group
  reorder   reorder_states: every layer's cached states moved to the beams that survived

Each case is a dict of plain values; ``prepare`` makes its inputs on the GPU from a seed,
``run`` is one call (in plain torch operations while ``own`` is false), ``exact`` the same
outputs in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
PAD_ID = 0
POWERS = tuple(2.0 ** e for e in range(-127, 128))  # tables: a library's log2 and pow may miss whole powers


# ---------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------

def _quantize(rows, cols, dtype):
    return {"kind": "quantize", "rows": rows, "cols": cols, "dtype": dtype}


def _product(rows, n, k, dtype, out, bias=False):
    return {"kind": "product", "rows": rows, "n": n, "k": k, "dtype": dtype, "out": out, "bias": bias}


def _select(groups, beams, vocab, count, dtype, masked=False, done=False):
    return {"kind": "select", "groups": groups, "beams": beams, "vocab": vocab, "count": count, "dtype": dtype,
            "masked": masked, "done": done}


def _reorder(groups, beams, states, heads, capacity, dim, shortest, longest, survivors, in_place):
    return {"kind": "reorder", "groups": groups, "beams": beams, "states": states, "heads": heads,
            "capacity": capacity, "dim": dim, "shortest": shortest, "longest": longest, "survivors": survivors,
            "in_place": in_place}


def _named(name, case):
    return {"name": name, **case}


def listed():
    return [
        # One token's hidden state to MXFP4 and back: latency.
        _named("quantize_token", _quantize(1, 896, "f32")),
        # An odd batch of wide activations whose rows end inside a block.
        _named("quantize_ragged_bf16", _quantize(1531, 4850, "bf16")),
        # A vocabulary's head converted when a model is loaded.
        _named("quantize_head_f16", _quantize(151936, 896, "f16")),
        # The last layer of one sequence's decode step.
        _named("logits_one_token", _product(1, 151936, 896, "f32", "f32")),
        # A small serving batch; rows and reduction that fill no tile.
        _named("logits_ragged24", _product(24, 50257, 800, "f16", "f32", bias=True)),
        # A layer's projection for drafted tokens or a short prompt.
        _named("project_prompt300", _product(300, 4864, 4096, "bf16", "bf16")),
        # A long prompt through a large layer: matrix work.
        _named("project_prompt4096", _product(4096, 16384, 8192, "bf16", "bf16")),
        # Beam search over one sequence.
        _named("select_one", _select(1, 4, 151936, 8, "f32")),
        # Constrained beam search on half-precision logits, some beams already ended.
        _named("select_masked_f16", _select(17, 4, 50257, 8, "f16", masked=True, done=True)),
        # A serving batch of beam searches.
        _named("select_batch", _select(64, 8, 151936, 16, "f32")),
        # The caches of one short sequence, moved where they lie.
        _named("reorder_one", _reorder(1, 4, 8, 2, 256, 64, 97, 97, 2, True)),
        # The caches of a batch of searches of different lengths, into the other set of buffers.
        _named("reorder_batch", _reorder(16, 4, 48, 2, 1024, 64, 1, 1024, 3, False)),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "select", "select", "reorder"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "quantize":
        rows, cols = _between(rng, 1, 4096), _between(rng, 64, 8192)
        return _quantize(rows, cols, dtype)
    if kind == "product":
        rows, n, k = _between(rng, 1, 2048), _between(rng, 256, 65536), 8 * _between(rng, 32, 1024)
        n = min(n, max(256, 2 ** 38 // (rows * k)))
        return _product(rows, n, k, dtype, rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.4)
    if kind == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        groups, vocab = _between(rng, 1, 256 // beams), _between(rng, 500, 151936)
        count = rng.choice([beams, 2 * beams, 2 * beams + 1])
        return _select(groups, beams, vocab, count, dtype, rng.random() < 0.4, rng.random() < 0.4)
    beams = rng.choice([2, 3, 4, 5, 8, 12, 16])
    groups, states = _between(rng, 1, max(1, 64 // beams)), 2 * _between(rng, 1, 24)
    capacity = _between(rng, 64, 1024)
    longest = rng.randint(1, capacity)
    in_place = rng.random() < 0.5
    survivors = rng.randint(1, beams - 1 if in_place else beams)
    return _reorder(groups, beams, states, rng.choice([1, 2, 3, 8]), capacity, rng.choice([40, 64, 128]),
                    rng.randint(1, longest), longest, survivors, in_place)


def _lengths(case):
    """The groups' lengths, from the shortest to the longest in equal steps."""
    steps = max(case["groups"] - 1, 1)
    span = case["longest"] - case["shortest"]
    return [case["shortest"] + span * g // steps for g in range(case["groups"])]


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    kind = case["kind"]
    if kind == "quantize":
        # Activations: normal, with a few channels much larger than the others.
        x = torch.randn(case["rows"], case["cols"], device="cuda", generator=g)
        x *= torch.exp(torch.randn(case["cols"], device="cuda", generator=g))
        state["x"] = x.to(DTYPES[case["dtype"]])
    elif kind == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        blocks = -(-k // BLOCK)
        x = torch.randn(rows, k, device="cuda", generator=g)
        state["x"] = x.to(DTYPES[case["dtype"]])
        # A checkpoint's weights: two codes to a byte, the lower column in the low half, and one
        # biased exponent to a block; what lies past the last column is zero.
        codes = torch.randint(0, 256, (n, blocks * BLOCK // 2), dtype=torch.uint8, device="cuda", generator=g)
        codes[:, (k + 1) // 2:] = 0
        if k % 2:
            codes[:, k // 2] &= 15
        scales = torch.randint(118, 123, (n, blocks), dtype=torch.uint8, device="cuda", generator=g)
        state["bias"] = torch.randn(n, device="cuda", generator=g) if case["bias"] else None
        if own:
            from tabby_amd import mx4
            state["head"] = mx4.LmHeadMx4(mx4.Mx4Matrix.from_rowmajor(codes, scales, k), bias=state["bias"])
        else:
            state["codes"], state["scales"] = codes, scales
    elif kind == "select":
        groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
        rows = groups * beams
        x = torch.randn(rows, vocab, device="cuda", generator=g) * 2.5
        hot = torch.randint(0, vocab, (rows, 8), device="cuda", generator=g)
        x.scatter_(1, hot, 9.0 + 4.0 * torch.rand(rows, 8, device="cuda", generator=g))
        state["logits"] = x.to(DTYPES[case["dtype"]])
        state["scores"] = -12.0 + 1.5 * torch.randn(groups, beams, device="cuda", generator=g)
        state["allowed"] = state["done"] = None
        if case["masked"]:
            # One bit to an entry: the low half of each word from one draw, the high half from another.
            words = -(-vocab // 32)
            low = torch.randint(0, 2 ** 16, (rows, words), device="cuda", generator=g)
            high = torch.randint(-2 ** 15, 2 ** 15, (rows, words), device="cuda", generator=g)
            state["allowed"] = (high * 2 ** 16 + low).to(torch.int32)
        if case["done"]:
            state["done"] = (torch.rand(groups, beams, device="cuda", generator=g) < 0.2).to(torch.int32)
        if own:
            from tabby_amd import beam
            state["selector"] = beam.BeamSelect(groups_max=groups, beams_max=beams, vocab_max=vocab,
                                                count_max=case["count"])
    else:
        groups, beams, survivors = case["groups"], case["beams"], case["survivors"]
        rows = groups * beams
        shape = (rows, case["heads"], case["capacity"], case["dim"])
        state["states"] = [torch.randn(shape, device="cuda", generator=g, dtype=torch.bfloat16)
                           for _ in range(case["states"])]
        order = torch.rand(groups, beams, device="cuda", generator=g).argsort(1)
        kept = order[:, :survivors]
        if case["in_place"]:
            # The survivors keep their slots and the others take a survivor's state.
            parents = torch.arange(beams, device="cuda").repeat(groups, 1)
            rest = beams - survivors
            source = kept.repeat(1, -(-rest // survivors))[:, :rest]
            parents.scatter_(1, order[:, survivors:], source)
        else:
            parents = kept.repeat(1, -(-beams // survivors))[:, :beams]
        state["parents"] = parents.to(torch.int32).contiguous()
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        state["out"] = None if case["in_place"] else [torch.zeros_like(s) for s in state["states"]]
    return state


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state, state["case"])
    return _PLAIN[kind](state, state["case"])


def _own_quantize(state, case):
    from tabby_amd import mx4
    return mx4.Mx4Matrix.quantize(state["x"]).dequantize(DTYPES[case["dtype"]])


def _own_product(state, case):
    return state["head"].logits(state["x"], dtype=DTYPES[case["out"]])


def _own_select(state, case):
    return tuple(state["selector"](state["logits"], state["scores"], case["count"], allowed=state["allowed"],
                                   done=state["done"], pad_id=PAD_ID))


def _own_reorder(state, case):
    from tabby_amd import beam
    return beam.reorder_states(state["states"], state["parents"], lengths=state["lengths"], out=state["out"])


def _round_blocks(x):
    """The values, in 32 bits, that the rows' blocks of 32 stand for once quantised."""
    rows, cols = x.shape
    pad = -cols % BLOCK
    v = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, BLOCK)
    amax = v.abs().amax(-1, keepdim=True)
    # frexp's mantissa lies in [1/2, 1): the power of two of the largest value is one below. The
    # largest code is 6 = 1.5 * 2^2.
    power = (torch.frexp(amax).exponent - 1 - 2).clamp(-127, 127)
    power = torch.where(amax > 0, power, torch.full_like(power, -127))
    scale = torch.tensor(POWERS, dtype=torch.float64, device=x.device)[power.long() + 127]
    a = v.double().abs() / scale
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp_max(6.0)
    out = torch.copysign(a * scale, v.double())
    out = torch.where(torch.isfinite(amax), out, torch.full_like(out, math.nan))
    return out.float().view(rows, -1)[:, :cols]


def _plain_quantize(state, case):
    return _round_blocks(state["x"]).to(DTYPES[case["dtype"]])


def _weights(codes, scales, k, dtype):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=dtype, device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1, BLOCK)
    w = table[both.int()] * torch.tensor(POWERS, dtype=dtype, device=codes.device)[scales.int()][:, :, None]
    return w.view(codes.shape[0], -1)[:, :k]


def _plain_product(state, case):
    w = _weights(state["codes"], state["scales"], case["k"], torch.float32)
    y = _round_blocks(state["x"]) @ w.t()
    if state["bias"] is not None:
        y = y + state["bias"]
    return y.to(DTYPES[case["out"]])


def _bits(words, vocab):
    """Truth values [rows, vocab] of a packed mask (entry t at bit t mod 32 of word t / 32)."""
    shifts = torch.arange(32, device=words.device, dtype=torch.int32)
    return ((words[:, :, None] >> shifts) & 1).bool().view(words.shape[0], -1)[:, :vocab]


def _plain_select(state, case):
    groups, beams, vocab, count = case["groups"], case["beams"], case["vocab"], case["count"]
    # The order of candidates of different beams hangs on their rows' sums: 64 bits.
    x = state["logits"].double()
    if state["allowed"] is not None:
        x = torch.where(_bits(state["allowed"], vocab), x, -math.inf)
    top = x.amax(1, keepdim=True)
    norm = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    score = state["scores"].double().view(-1, 1) + (x - norm)
    if state["done"] is not None:
        ended = state["done"].view(-1, 1) != 0
        at_pad = torch.arange(vocab, device=x.device) == PAD_ID
        kept = torch.where(at_pad, state["scores"].double().view(-1, 1), -math.inf)
        score = torch.where(ended, kept, score)
    best, at = torch.sort(score.view(groups, -1), dim=1, descending=True, stable=True)
    best, at = best[:, :count], at[:, :count]
    none = best == -math.inf
    tokens = torch.where(none, -1, at % vocab).int()
    parents = torch.where(none, -1, at // vocab).int()
    return tokens, parents, best.float()


def _plain_reorder(state, case):
    groups, beams = case["groups"], case["beams"]
    base = torch.arange(groups, device="cuda")[:, None] * beams
    source = (base + state["parents"]).view(-1)
    position = torch.arange(case["capacity"], device="cuda")
    used = (position[None] < state["lengths"][:, None]).repeat_interleave(beams, 0)[:, None, :, None]
    out = state["out"] or state["states"]
    for s, o in zip(state["states"], out):
        o.copy_(torch.where(used, s[source], o))
    return out


_OWN = {"quantize": _own_quantize, "product": _own_product, "select": _own_select, "reorder": _own_reorder}
_PLAIN = {"quantize": _plain_quantize, "product": _plain_product, "select": _plain_select,
          "reorder": _plain_reorder}


# ---------------------------------------------------------------------------------------
# What a pass cannot do without, and its outputs in 64 bits
# ---------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "quantize":
        size = case["rows"] * case["cols"]
        held = size / 2 + case["rows"] * -(-case["cols"] // BLOCK)
        return {"bytes": 2 * size * SIZES[case["dtype"]] + 2 * held, "flops": 4.0 * size}
    if kind == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        held = n * k / 2 + n * -(-k // BLOCK)
        moved = rows * k * SIZES[case["dtype"]] + rows * n * SIZES[case["out"]] + (4 * n if case["bias"] else 0)
        return {"bytes": held + moved, "flops": 2.0 * rows * n * k}
    if kind == "select":
        rows, vocab = case["groups"] * case["beams"], case["vocab"]
        read = rows * vocab * SIZES[case["dtype"]] + (rows * -(-vocab // 32) * 4 if case["masked"] else 0)
        return {"bytes": read + 4 * rows + 12 * case["groups"] * case["count"], "flops": 4.0 * rows * vocab}
    survivors, beams = case["survivors"], case["beams"]
    if case["in_place"]:
        moved = beams - survivors + min(survivors, beams - survivors)
    else:
        moved = beams + survivors
    each = case["states"] * case["heads"] * case["dim"] * 2
    return {"bytes": each * moved * sum(_lengths(case)), "flops": 0.0}


def _nearest(x):
    """Values in 64 bits of the quantised rows: the code by comparisons with the midpoints."""
    rows, cols = x.shape
    v = torch.zeros(rows, -(-cols // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    v[:, :cols] = x.double()
    out = torch.empty_like(v)
    levels = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    powers = torch.tensor(POWERS, dtype=torch.float64, device=x.device)
    for c in range(0, v.shape[1], BLOCK):
        block = v[:, c:c + BLOCK]
        largest = block.abs().max(1, keepdim=True).values
        # The largest power of two that is no larger than a quarter of the largest value.
        power = powers[(torch.searchsorted(powers, largest / 4, right=True) - 1).clamp(0, 254)]
        a = (block / power).abs()
        code = torch.zeros_like(a, dtype=torch.int64)
        for j in range(7):
            middle = (E2M1[j] + E2M1[j + 1]) / 2
            code += (a > middle) if j % 2 == 0 else (a >= middle)
        value = torch.sign(block) * levels[code] * power
        out[:, c:c + BLOCK] = torch.where(torch.isfinite(largest), value, math.nan)
    return out[:, :cols]


def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    kind = case["kind"]
    if kind == "quantize":
        return _nearest(state["x"])
    if kind == "product":
        k, codes = case["k"], state["codes"]
        low, high = (codes & 15).long(), (codes >> 4).long()
        levels = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
        w = torch.empty(case["n"], 2 * codes.shape[1], dtype=torch.float64, device="cuda")
        for half, part in ((0, low), (1, high)):
            w[:, half::2] = levels[part & 7] * (1 - 2 * (part >> 3))
        w *= torch.tensor(POWERS, dtype=torch.float64, device="cuda")[state["scales"].long()].repeat_interleave(BLOCK, 1)
        y = torch.mm(_nearest(state["x"]), w[:, :k].t().contiguous())
        return y if state["bias"] is None else y + state["bias"].double()
    if kind == "select":
        return _best(state, case)
    out = state["out"] or [s.clone() for s in state["states"]]
    parents, lengths = state["parents"].tolist(), _lengths(case)
    for s, o in zip(state["states"], out):
        old = s.clone() if o is s else s
        for g, length in enumerate(lengths):
            for b, parent in enumerate(parents[g]):
                o[g * case["beams"] + b, :, :length] = old[g * case["beams"] + parent, :, :length]
    return out


def _best(state, case):
    """Each beam's own best entries, then each group's best of those."""
    groups, beams, vocab, count = case["groups"], case["beams"], case["vocab"], case["count"]
    take = min(count, vocab)
    tokens = torch.full((groups, count), -1, dtype=torch.int32, device="cuda")
    parents = tokens.clone()
    scores = torch.full((groups, count), -math.inf, dtype=torch.float64, device="cuda")
    cumulative = state["scores"].double()
    for g in range(groups):
        found = []
        for b in range(beams):
            r = g * beams + b
            if state["done"] is not None and int(state["done"][g, b]):
                found.append((cumulative[g, b].view(1), torch.tensor([PAD_ID], device="cuda"), b))
                continue
            row = state["logits"][r].double()
            if state["allowed"] is not None:
                bit = torch.arange(vocab, device="cuda")
                row = row.masked_fill((state["allowed"][r].long()[bit // 32] >> (bit % 32)) & 1 == 0, -math.inf)
            values, ids = torch.sort(row, descending=True, stable=True)
            lead = values[:take] - torch.logsumexp(row, 0)
            found.append((cumulative[g, b] + lead, ids[:take], b))
        value = torch.cat([f[0] for f in found])
        token = torch.cat([f[1] for f in found])
        parent = torch.cat([torch.full_like(f[1], f[2]) for f in found])
        flat = parent * vocab + token
        order = torch.argsort(flat)
        order = order[torch.sort(value[order], descending=True, stable=True).indices][:count]
        order = order[value[order] > -math.inf]
        n = order.numel()
        tokens[g, :n], parents[g, :n] = token[order].int(), parent[order].int()
        scores[g, :n] = value[order]
    return tokens, parents, scores
