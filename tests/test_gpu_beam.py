"""Beam search's selection and reordering against a plain restatement in 64 bits: tokens,
parents and states exactly, scores within the rounding of their type."""
import numpy as np
import pytest

from tabby_amd import sampler as S

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16"]
INF = float("inf")


def _torch():
    import torch
    assert torch.cuda.is_available(), "needs an MI355X"
    return torch


def _beam():
    from tabby_amd import beam
    return beam


def _dtype(name):
    torch = _torch()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def choose(logits, scores, count, allowed=None, done=None, pad=0):
    """(tokens, parents, scores, status) of every group, in float64."""
    groups, beams = scores.shape
    tokens = np.full((groups, count), -1, dtype=np.int32)
    parents = tokens.copy()
    best = np.full((groups, count), -INF)
    status = np.zeros(groups, dtype=np.int32)
    for g in range(groups):
        found = []
        for b in range(beams):
            s = float(scores[g, b])
            if np.isnan(s) or s == INF:
                status[g] = S.TABBY_EDOMAIN
                continue
            if s == -INF:
                continue
            if done is not None and done[g, b]:
                found.append((-s, b, pad))
                continue
            x = logits[g * beams + b].astype(np.float64)
            ids = np.arange(x.size) if allowed is None else np.nonzero(allowed[g * beams + b])[0]
            x = x[ids]
            if np.isnan(x).any() or (x == INF).any():
                status[g] = S.TABBY_EDOMAIN
                continue
            keep = x > -INF
            x, ids = x[keep], ids[keep]
            if x.size == 0:
                continue
            m = x.max()
            norm = m + np.log(np.sum(np.exp(x - m)))
            order = np.lexsort((ids, -x))[:count]
            found += [(-(s + (x[i] - norm)), b, int(ids[i])) for i in order]
        if status[g]:
            continue
        if not found:
            status[g] = S.TABBY_EEMPTY
        for j, (v, b, t) in enumerate(sorted(found)[:count]):
            tokens[g, j], parents[g, j], best[g, j] = t, b, -v
    return tokens, parents, best, status


def _check(logits, scores, count, allowed=None, done=None, pad=0, ctx=""):
    """`logits` a CUDA tensor; the rest numpy (allowed: truth values)."""
    torch = _torch()
    beam = _beam()
    groups, beams = scores.shape
    vocab = logits.shape[1]
    sel = beam.BeamSelect(vocab_max=vocab, groups_max=groups, beams_max=beams, count_max=count)
    status = torch.full((groups,), -5, dtype=torch.int32, device="cuda")
    print(f"select {groups} x {beams} x {vocab} keep {count} {logits.dtype} {ctx}", flush=True)
    got = sel(logits, torch.from_numpy(scores.astype(np.float32)).cuda(), count,
              allowed=None if allowed is None else beam.pack_mask(torch.from_numpy(allowed)).cuda(),
              done=None if done is None else torch.from_numpy(done.astype(np.int32)).cuda(), pad_id=pad, status=status)
    want = choose(logits.double().cpu().numpy(), scores.astype(np.float32), count, allowed, done, pad)
    assert np.array_equal(status.cpu().numpy(), want[3]), ctx
    assert np.array_equal(got.tokens.cpu().numpy(), want[0]), (ctx, got.tokens.cpu().numpy(), want[0])
    assert np.array_equal(got.parents.cpu().numpy(), want[1]), ctx
    have = got.scores.double().cpu().numpy()
    real = want[2] > -INF
    assert np.array_equal(have > -INF, real), ctx
    # Half a step of f32; a row's logarithm may come from f32 exponentials (2^-21 of the sum).
    err = np.abs(have[real] - want[2][real])
    assert (err <= 2.0 ** -24 * np.abs(want[2][real]) + 2.0 ** -21).all(), (ctx, err.max())
    return got


def _logits(rows, vocab, dtype, seed, sigma=2.5, spikes=True):
    torch = _torch()
    rng = np.random.default_rng(seed)
    x = rng.normal(0, sigma, (rows, vocab))
    if spikes:
        for r in range(rows):
            x[r, rng.integers(0, vocab, min(8, vocab))] = rng.uniform(9, 13, min(8, vocab))
    return torch.from_numpy(x).to(_dtype(dtype)).cuda()


def _scores(groups, beams, seed):
    return np.random.default_rng(seed).normal(-12, 1.5, (groups, beams)).astype(np.float32)


@pytest.mark.parametrize("groups,beams,vocab,count", [
    (1, 1, 1, 1), (1, 1, 1, 5), (2, 3, 2, 4), (1, 4, 31, 8), (3, 2, 32, 4), (2, 2, 33, 128), (1, 4, 151936, 8),
    (5, 3, 1023, 6), (2, 4, 1024, 8), (2, 4, 1025, 9), (17, 4, 5003, 8), (3, 8, 16385, 16), (2, 16, 32000, 33),
    (1, 64, 4096, 128), (40, 5, 777, 10), (70, 8, 2048, 16), (1, 1, 151936, 128), (2, 64, 300, 128), (130, 2, 20001, 4),
    (300, 1, 3000, 2)])
def test_selection(groups, beams, vocab, count):
    dtype = TYPES[(groups + beams + vocab + count) % 3]
    _check(_logits(groups * beams, vocab, dtype, vocab + beams), _scores(groups, beams, vocab), count)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups,beams,vocab,count", [(1, 4, 50257, 8), (12, 4, 50257, 8), (64, 4, 9999, 4), (3, 5, 200, 11)])
def test_types_masks_and_ended_beams(dtype, groups, beams, vocab, count):
    rng = np.random.default_rng(groups * vocab)
    x = _logits(groups * beams, vocab, dtype, 3)
    allowed = rng.random((groups * beams, vocab)) < 0.4
    done = rng.random((groups, beams)) < 0.3
    s = _scores(groups, beams, 4)
    _check(x, s, count, allowed=allowed, ctx="mask")
    _check(x, s, count, done=done, pad=7, ctx="done")
    _check(x, s, count, allowed=allowed, done=done, pad=vocab + 3, ctx="both")


@pytest.mark.parametrize("vocab", [65, 5000, 40000])
def test_what_is_not_allowed_is_not_looked_at(vocab):
    torch = _torch()
    rng = np.random.default_rng(vocab)
    for dtype in TYPES:
        x = _logits(6, vocab, dtype, 8)
        allowed = rng.random((6, vocab)) < 0.5
        bad = torch.from_numpy(np.where(rng.random((6, vocab)) < 0.5, np.nan, INF)).to(x.dtype).cuda()
        y = torch.where(torch.from_numpy(allowed).cuda(), x, bad)
        s = _scores(2, 3, 1)
        got = _check(y, s, 7, allowed=allowed, ctx="nan outside")
        plain = _check(torch.where(torch.from_numpy(allowed).cuda(), x, torch.full_like(x, -INF)), s, 7, ctx="-inf instead")
        assert torch.equal(got.tokens, plain.tokens)
        low = torch.finfo(x.dtype).min
        _check(torch.where(torch.from_numpy(allowed).cuda(), x, torch.full_like(x, low)), s, 7, ctx="lowest value")


def test_rows_with_nothing_and_groups_with_nothing():
    torch = _torch()
    x = _logits(12, 700, "f32", 2)
    allowed = np.ones((12, 700), dtype=bool)
    allowed[1] = False            # one row of the first group
    allowed[3:6] = False          # the whole second group
    x[7] = -INF                   # a row of the third group holds only -inf
    s = _scores(4, 3, 5)
    s[2, 2] = -INF                # and another beam of it is dead
    s[3] = -INF                   # the fourth group is dead
    _check(x, s, 8, allowed=allowed)
    few = np.zeros((12, 700), dtype=bool)
    few[:, 690:692] = True        # fewer continuations than are kept
    _check(x, s, 8, allowed=few)


@pytest.mark.parametrize("vocab", [100, 30000])
def test_values_out_of_domain_spoil_their_group_alone(vocab):
    x = _logits(15, vocab, "f32", 12)
    x[4, vocab - 1] = float("nan")
    x[7, 3] = INF
    s = _scores(5, 3, 6)
    s[3, 1] = np.nan
    s[4, 0] = INF
    _check(x, s, 6)
    # In a beam that is not read they do no harm.
    done = np.zeros((5, 3))
    done[1, 1] = 1                # row 4
    dead = s.copy()
    dead[2, 1] = -INF             # row 7
    dead[3, 1] = dead[4, 0] = -10.0
    _check(x, dead, 6, done=done)


@pytest.mark.parametrize("groups,beams,vocab,count", [(1, 4, 1000, 8), (2, 4, 60000, 8), (300, 2, 500, 5), (2, 8, 20000, 128)])
def test_ties_go_to_the_lower_beam_and_token(groups, beams, vocab, count):
    torch = _torch()
    rng = np.random.default_rng(count)
    # Coarse logits, all of a group's beams alike and at one score: every value ties, in the row and across.
    row = np.round(rng.normal(0, 2, (groups, 1, vocab)) * 2) / 2
    x = torch.from_numpy(np.broadcast_to(row, (groups, beams, vocab)).reshape(-1, vocab).copy()).float().cuda()
    _check(x, np.full((groups, beams), -3.0, dtype=np.float32), count, ctx="alike")
    _check(torch.zeros_like(x), np.full((groups, beams), -3.0, dtype=np.float32), count, ctx="constant")


def test_first_step_has_one_live_beam():
    x = _logits(8, 5000, "bf16", 30)
    s = np.full((2, 4), -INF, dtype=np.float32)
    s[:, 0] = 0.0
    _check(x, s, 4)


def test_peaked_and_flat_rows():
    torch = _torch()
    x = torch.zeros(4, 20000, device="cuda")
    x[1, 17] = 200.0              # everything else underflows
    x[2] = torch.linspace(-80, 0, 20000, device="cuda")
    x[3] = 3.0e38
    _check(x, np.array([[-1.0, -2.0, -3.0, -4.0]], dtype=np.float32), 9)
    _check(x - 3.0e38, np.array([[-1.0, -2.0, -3.0, -4.0]], dtype=np.float32), 9)


@pytest.mark.parametrize("order", ["ascending", "descending", "block"])
@pytest.mark.parametrize("vocab", [6000, 151936])
def test_rows_in_an_awkward_order(order, vocab):
    # The largest values last, first, or all together: a bound taken from a part of the row is poor.
    torch = _torch()
    rng = np.random.default_rng(vocab)
    x = np.sort(rng.normal(0, 3, (4, vocab)).astype(np.float32), axis=1)
    if order == "descending":
        x = x[:, ::-1]
    if order == "block":
        x = np.roll(x, vocab // 3, axis=1)
    _check(torch.from_numpy(x.copy()).cuda(), _scores(2, 2, 1), 128, ctx=order)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_apart_and_unaligned(dtype):
    torch = _torch()
    wide = _logits(6, 3003, dtype, 55)
    for lo, hi in ((0, 3000), (1, 2500), (3, 3003), (8, 2056)):
        _check(wide[:, lo:hi], _scores(2, 3, lo), 7, ctx=f"columns {lo}..{hi}")


def test_runs_alike_and_on_another_stream():
    torch = _torch()
    beam = _beam()
    x = _logits(96, 50257, "f16", 70)
    s = torch.from_numpy(_scores(24, 4, 2)).cuda()
    sel = beam.BeamSelect(vocab_max=50257, groups_max=24, beams_max=4, count_max=8)
    first = sel(x, s, 8)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    other = sel(x, s, 8, stream=side)
    side.synchronize()
    for a, b in zip(first, other):
        assert torch.equal(a, b)


def test_selection_in_a_graph():
    torch = _torch()
    beam = _beam()
    sel = beam.BeamSelect(vocab_max=9001, groups_max=3, beams_max=4, count_max=8)
    x, s = _logits(12, 9001, "f32", 80), torch.from_numpy(_scores(3, 4, 9)).cuda()
    sel(x, s, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = sel(x, s, 8)
    for seed in range(4):
        x.copy_(_logits(12, 9001, "f32", 200 + seed))
        graph.replay()
        torch.cuda.synchronize()
        now = sel(x, s, 8)
        for a, b in zip(held, now):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_selection_refusals():
    torch = _torch()
    beam = _beam()
    sel = beam.BeamSelect(vocab_max=100, groups_max=2, beams_max=4, count_max=8)
    x, s = torch.zeros(8, 100, device="cuda"), torch.zeros(2, 4, device="cuda")
    with pytest.raises(ValueError, match="8 rows"):
        sel(x, s[:1], 4)
    with pytest.raises(ValueError, match="exceed"):
        sel(torch.zeros(8, 101, device="cuda"), s, 4)
    with pytest.raises(ValueError, match="exceed"):
        sel(x, s, 9)
    with pytest.raises(ValueError, match="count"):
        sel(x, s, 0)
    with pytest.raises(ValueError, match="scores"):
        sel(x, s.double(), 4)
    with pytest.raises(ValueError, match="allowed"):
        sel(x, s, 4, allowed=torch.zeros(8, 3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="done"):
        sel(x, s, 4, done=torch.zeros(2, 4, device="cuda"))
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        sel(x.double(), s, 4)
    with pytest.raises(S.SamplingError, match="pad_id"):
        sel(x, s, 4, pad_id=-1)


# ---------------------------------------------------------------------------------------
# Reordering
# ---------------------------------------------------------------------------------------

def _moved(old, into, parents, lengths, position):
    """numpy: what every row of `into` becomes."""
    groups, beams = parents.shape
    new = into.copy()
    for g in range(groups):
        n = old.shape[position] if lengths is None else min(max(int(lengths[g]), 0), old.shape[position])
        for b in range(beams):
            p = int(parents[g, b])
            if 0 <= p < beams:
                at = (g * beams + b,) + (slice(None),) * (position - 1) + (slice(0, n),)
                src = (g * beams + p,) + (slice(None),) * (position - 1) + (slice(0, n),)
                new[at] = old[src]
    return new


def _check_reorder(shape, groups, beams, dtype="int16", states=3, in_place=True, lengths=None, seed=0, parents=None):
    torch = _torch()
    rng = np.random.default_rng(seed)
    info = np.iinfo(dtype)
    old = [rng.integers(info.min, info.max, shape, dtype=dtype) for _ in range(states)]
    into = old if in_place else [rng.integers(info.min, info.max, shape, dtype=dtype) for _ in range(states)]
    if parents is None:
        parents = rng.integers(-1, beams, (groups, beams)).astype(np.int32)
    print(f"reorder {shape} {groups} x {beams} {dtype} in_place={in_place} lengths={lengths}", flush=True)
    src = [torch.from_numpy(o).cuda() for o in old]
    out = None if in_place else [torch.from_numpy(o).cuda() for o in into]
    got = _beam().reorder_states(src, torch.from_numpy(parents).cuda(),
                                 lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                                 out=out)
    position = 2 if len(shape) == 4 else 1
    for i, t in enumerate(got):
        assert np.array_equal(t.cpu().numpy(), _moved(old[i], into[i], parents, lengths, position)), i
        if not in_place:
            assert np.array_equal(src[i].cpu().numpy(), old[i])


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("groups,beams,rest", [
    (1, 1, (1,)), (1, 4, (7,)), (2, 3, (5, 3)), (3, 4, (2, 16, 64)), (1, 5, (3, 100, 40)), (2, 8, (1, 33, 8)), (4, 12, (2, 9, 24)),
    (1, 16, (2, 50, 64)), (2, 17, (300, 4)), (1, 33, (2, 11, 20)), (1, 64, (2, 130, 16)), (5, 2, (1, 1, 1))])
def test_reorder(groups, beams, rest, in_place):
    for i, dtype in enumerate(("int8", "int16", "int32", "int64")):
        _check_reorder((groups * beams,) + rest, groups, beams, dtype, in_place=in_place, seed=beams + i)


@pytest.mark.parametrize("in_place", [True, False])
def test_reorder_lengths(in_place):
    _check_reorder((20, 3, 70, 48), 5, 4, in_place=in_place, lengths=[0, 1, 70, 69, 33])
    _check_reorder((12, 40, 64), 3, 4, in_place=in_place, lengths=[-7, 1000, 17])  # held to the capacity
    _check_reorder((12, 97), 3, 4, "int32", in_place=in_place, lengths=[96, 2, 5])


def test_reorder_cycles_and_copies_in_place():
    for p in ([1, 2, 3, 0], [3, 2, 1, 0], [0, 0, 0, 0], [1, 0, 1, 0], [2, 2, 3, 3], [0, 1, 2, 3], [-1, 0, 4, 99], [-1, -1, -1, -1]):
        _check_reorder((8, 2, 37, 64), 2, 4, parents=np.array([p, p[::-1]], dtype=np.int32))


def test_reorder_many_states():
    _check_reorder((8, 2, 20, 16), 2, 4, states=131)
    _check_reorder((8, 2, 20, 16), 2, 4, states=65, in_place=False)


def test_reorder_views_and_what_lies_beside_them():
    torch = _torch()
    rng = np.random.default_rng(4)
    base = rng.integers(0, 30000, (8, 3, 50, 64), dtype=np.int16)
    parents = np.array([[1, 1, 3, 2], [0, 0, 0, 1]], dtype=np.int32)
    for seg, lo, hi in ((slice(0, 3), 0, 30), (slice(1, 3), 10, 50), (slice(0, 1), 3, 4)):
        t = torch.from_numpy(base).cuda()
        _beam().reorder_states([t[:, seg, lo:hi]], torch.from_numpy(parents).cuda())
        want = base.copy()
        want[:, seg, lo:hi] = _moved(base[:, seg, lo:hi], base[:, seg, lo:hi], parents, None, 2)
        assert np.array_equal(t.cpu().numpy(), want)
    odd = torch.from_numpy(base.reshape(8, -1)).cuda()
    _beam().reorder_states([odd[:, 1:1000]], torch.from_numpy(parents).cuda())
    want = base.reshape(8, -1).copy()
    want[:, 1:1000] = _moved(want[:, 1:1000], want[:, 1:1000], parents, None, 1)
    assert np.array_equal(odd.cpu().numpy(), want)


def test_reorder_past_32_bits():
    # Two rows more than 4 GiB apart: the addresses need 64 bits.
    torch = _torch()
    t = torch.zeros((4, 2 ** 31 + 64), dtype=torch.uint8, device="cuda")
    for b in range(4):
        t[b, :64] = b + 1
        t[b, -64:] = 10 * (b + 1)
    _beam().reorder_states([t], torch.tensor([[3, 0, 0, 2]], dtype=torch.int32, device="cuda"))
    assert t[:, 0].tolist() == [4, 1, 1, 3] and t[:, -1].tolist() == [40, 10, 10, 30]
    assert int(t[:, 64:-64].max()) == 0


def test_selection_past_32_bits():
    torch = _torch()
    x = torch.zeros((2, 2 ** 31 + 8), dtype=torch.float16, device="cuda")
    view = x[:, 5:40005]
    view.copy_(_logits(2, 40000, "f16", 5))
    _check(view, _scores(1, 2, 3), 4)


def test_reorder_in_a_graph():
    torch = _torch()
    beam = _beam()
    states = [torch.randint(0, 30000, (8, 2, 40, 64), dtype=torch.int16, device="cuda") for _ in range(4)]
    out = [torch.zeros_like(s) for s in states]
    parents = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    lengths = torch.tensor([40, 11], dtype=torch.int32, device="cuda")
    beam.reorder_states(states, parents, lengths=lengths, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        beam.reorder_states(states, parents, lengths=lengths, out=out)
    for i in range(4):
        parents.copy_(torch.tensor([[i, 0, 1, 3], [3 - i, 2, 2, -1]], dtype=torch.int32))
        before = [o.cpu().numpy() for o in out]
        graph.replay()
        torch.cuda.synchronize()
        for s, o, b in zip(states, out, before):
            assert np.array_equal(o.cpu().numpy(), _moved(s.cpu().numpy(), b, parents.cpu().numpy(), [40, 11], 2))


def test_reorder_refusals():
    torch = _torch()
    beam = _beam()
    t = torch.zeros(8, 2, 10, 4, device="cuda")
    p = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="empty"):
        beam.reorder_states([], p)
    with pytest.raises(ValueError, match="int32"):
        beam.reorder_states([t], p.long())
    with pytest.raises(ValueError, match="8 rows"):
        beam.reorder_states([t[:4]], p)
    with pytest.raises(ValueError, match="one after another"):
        beam.reorder_states([t.transpose(2, 3)], p)
    with pytest.raises(ValueError, match="one shape"):
        beam.reorder_states([t, t[:, :1]], p)
    with pytest.raises(ValueError, match="laid out"):
        beam.reorder_states([t], p, out=[torch.zeros(8, 2, 11, 4, device="cuda")])
    with pytest.raises(ValueError, match="lengths"):
        beam.reorder_states([t], p, lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="device"):
        beam.reorder_states([t.cpu()], p)
    with pytest.raises(S.SamplingError, match="overlap"):
        wide = torch.zeros(8, 2, 12, 4, device="cuda")
        beam.reorder_states([wide[:, :, :10]], p, out=[wide[:, :, 1:11]])


# ---------------------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------------------

def test_search_finds_what_a_plain_search_finds():
    # A chain over few tokens: its states are the tokens so far, so the plain search needs none.
    torch = _torch()
    beam = _beam()
    vocab, beams, steps, groups, end = 23, 3, 7, 4, 5
    rng = np.random.default_rng(6)
    table = rng.normal(0, 2, (groups, vocab, vocab)).astype(np.float32)
    start = rng.integers(0, vocab, groups)
    search = beam.BeamSearch(groups, beams, vocab, steps, end_ids=(end,), pad_id=0)
    dev = torch.from_numpy(table).cuda()
    last = torch.from_numpy(np.repeat(start, beams)).cuda()
    history = torch.zeros((groups * beams, steps, 4), dtype=torch.int32, device="cuda")
    group = torch.arange(groups, device="cuda").repeat_interleave(beams)
    for i in range(steps):
        last = search.step(dev[group, last.long()].contiguous(), states=[history])
        history[:, i] = last[:, None]
    for g in range(groups):
        live = [(0.0, (), False)]
        for _ in range(steps):
            grown = []
            for b, (s, ids, ended) in enumerate(live):
                if ended:
                    grown.append((-s, b, 0, True))
                    continue
                row = table[g, ids[-1] if ids else start[g]].astype(np.float64)
                lp = row - (row.max() + np.log(np.exp(row - row.max()).sum()))
                grown += [(-(s + lp[t]), b, t, t == end) for t in range(vocab)]
            live = [(float(np.float32(-v)), live[b][1] + (t,), e) for v, b, t, e in sorted(grown)[:beams]]
        rows = slice(g * beams, (g + 1) * beams)
        assert search.tokens[rows].tolist() == [list(l[1]) for l in live]
        assert np.allclose(search.scores[g].cpu().numpy(), [l[0] for l in live], rtol=0, atol=1e-4)
        assert torch.equal(history[rows, :, 0], search.tokens[rows])
        assert search.done[g].tolist() == [int(l[2]) for l in live]
    assert len(search.best()) == groups


def test_example_runs_the_product_the_selection_and_the_states_together():
    # examples/beam_search_mx4.py against a plain search in 64 bits over the values its head stands for.
    import os
    import sys
    torch = _torch()
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import beam_search_mx4 as example
    import mx4_oracle as M
    vocab, hidden, beams, steps = 397, 160, 3, 6
    model = example.Model(vocab, hidden, seed=3)
    prompt = torch.tensor([5, 77, 396], dtype=torch.int32, device="cuda")
    best, run = example.search(model, prompt, beams, steps, end_ids=(9,))
    weight = model.head.weight.dequantize().double().cpu().numpy()
    embed = model.embed.cpu()
    for g, first in enumerate(prompt.tolist()):
        live = [(0.0, (), False, [])]
        for _ in range(steps):
            grown = []
            for b, (s, ids, ended, kept) in enumerate(live):
                h = embed[ids[-1] if ids else first]
                if kept:
                    h = h + torch.stack(kept).float().mean(0)
                kept = kept + [h.to(torch.bfloat16)]
                if ended:
                    grown.append((-s, b, 0, True, kept))
                    continue
                row = M.rounded(h.double().numpy()[None])[0] @ weight.T
                lp = row - (row.max() + np.log(np.exp(row - row.max()).sum()))
                grown += [(-(s + lp[t]), b, t, t == 9, kept) for t in range(vocab)]
            grown.sort(key=lambda v: v[:3])
            live = [(float(np.float32(-v)), live[b][1] + (t,), e, kept) for v, b, t, e, kept in grown[:beams]]
        assert run.tokens[g * beams:(g + 1) * beams].tolist() == [list(l[1]) for l in live]
        assert np.allclose(run.scores[g].cpu().numpy(), [l[0] for l in live], rtol=0, atol=1e-3)
        stop = next((i + 1 for i, t in enumerate(live[0][1]) if t == 9), steps)
        assert best[g][0] == list(live[0][1])[:stop]


def test_a_failed_group_keeps_its_first_failure():
    torch = _torch()
    search = _beam().BeamSearch(3, 2, 50, 4)
    x = _logits(6, 50, "f32", 1)
    search.step(x)
    x[2, 7] = float("nan")
    search.step(x)
    search.step(_logits(6, 50, "f32", 2))
    assert search.status.tolist() == [0, S.TABBY_EDOMAIN, 0]
    with pytest.raises(S.SamplingError, match="group 1: a logit or score"):
        search.best()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups,beams,vocab,count", [
    (1, 1, 262143, 64), (1, 2, 151936, 40), (2, 64, 9000, 128), (1, 16, 151936, 32), (3, 33, 8193, 17), (65, 4, 12289, 65),
    (40, 8, 40961, 33), (260, 1, 4097, 128), (9, 2, 60000, 3)])
def test_parts_waves_and_merges(groups, beams, vocab, count, dtype):
    # Every shape of workgroup, of parts to a row (with the last one short) and of merge.
    _check(_logits(groups * beams, vocab, dtype, vocab + count), _scores(groups, beams, count), count)


@pytest.mark.parametrize("count", [7, 32, 33, 64, 65, 128])
def test_ascending_rows_fill_the_lists(count):
    # Every chunk lies above every bound that came before it: the lists overflow and the row is read again.
    torch = _torch()
    rows = []
    for step in (1e-4, 3e-3):
        rows += [np.arange(70000) * step, np.arange(70000) // 64 * step]
    x = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda()
    _check(x, _scores(2, 2, count), count)
    _check(x.repeat(80, 1), _scores(160, 2, count), count)


def test_equal_rows_score_alike():
    # The sums do not hang on the order in which waves and workgroups end: equal rows tie to the last bit.
    torch = _torch()
    x = _logits(1, 100003, "f32", 9).repeat(320, 1)
    s = np.full((40, 8), -1.0, dtype=np.float32)
    got = _check(x, s, 16, ctx="equal rows")
    assert (got.scores == got.scores[:1]).all() and (got.tokens == got.tokens[:1]).all()


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("beams", [7, 15, 31, 40, 63])
def test_reorder_many_beams_of_wide_columns(beams, in_place):
    _check_reorder((2 * beams, 2, 19, 128), 2, beams, in_place=in_place, lengths=[19, 6], seed=beams)
    _check_reorder((2 * beams, 5, 24), 2, beams, "int8", in_place=in_place, seed=beams)
    _check_reorder((2 * beams, 37), 2, beams, "int32", in_place=in_place, seed=beams)


@pytest.mark.parametrize("seed", range(6))
def test_reorder_states_in_one_buffer(seed):
    # Views of one buffer, side by side or across each other: refused if they share an element that is written, and
    # moved like states of their own if not.
    torch = _torch()
    rng = np.random.default_rng(seed)
    moved = refused = 0
    for trial in range(60):
        groups, beams = int(rng.integers(1, 3)), int(rng.integers(1, 4))
        rows, segments, positions, width = groups * beams, int(rng.integers(1, 4)), int(rng.integers(1, 4)), int(rng.integers(1, 5))
        segment = positions * width
        segment_stride = segment * int(rng.integers(1, 4))
        extent = (segments - 1) * segment_stride + segment
        row_stride = extent + int(rng.choice([0, 0, segment, extent, 2 * extent]))
        span = (rows - 1) * row_stride + extent
        n, in_place = int(rng.integers(2, 5)), bool(rng.integers(0, 2))
        step = int(rng.choice([segment, extent, row_stride, span]))
        count = n if in_place else 2 * n
        offsets = rng.permutation(count * 2)[:count] * step
        if trial % 3 == 0:
            offsets = offsets + rng.integers(-1, 2, count) * (rng.random(count) < 0.3)
        offsets = offsets - offsets.min()
        base = rng.integers(0, 30000, int(offsets.max()) + span + 8, dtype=np.int16)
        shape, strides = (rows, segments, positions, width), (row_stride, segment_stride, width, 1)
        at = np.zeros(shape, dtype=np.int64)
        for axis, stride in enumerate(strides):
            at += (np.arange(shape[axis]) * stride).reshape([-1 if i == axis else 1 for i in range(4)])
        buffer = torch.from_numpy(base).cuda()
        views = [torch.as_strided(buffer, shape, strides, int(o)) for o in offsets]
        parents = rng.integers(-1, beams, (groups, beams)).astype(np.int32)
        src, out = (views, None) if in_place else (views[:n], views[n:])
        owners = np.zeros(base.size, dtype=np.int64)
        for o in offsets if in_place else offsets[n:]:
            owners[at + o] += 1
        clash = (owners > 1).any() or (not in_place and any((owners[at + o] > 0).any() for o in offsets[:n]))
        print(f"one buffer {shape} {strides} at {offsets.tolist()} in_place={in_place} clash={clash}", flush=True)
        if clash:
            refused += 1
            with pytest.raises(S.SamplingError, match="overlap"):
                _beam().reorder_states(src, torch.from_numpy(parents).cuda(), out=out)
            continue
        moved += 1
        _beam().reorder_states(src, torch.from_numpy(parents).cuda(), out=out)
        want = base.copy()
        for i in range(n):
            to = at + (offsets[i] if in_place else offsets[n + i])
            want[to] = _moved(base[at + offsets[i]], base[to], parents, None, 2)
        assert np.array_equal(buffer.cpu().numpy(), want)
    assert moved > 5 and refused > 5


def test_a_search_on_another_stream():
    # Step by step on the current stream and on one of its own, which ends while the current one is busy.
    torch = _torch()
    beam = _beam()
    steps = [_logits(6, 4001, "f32", 40 + i) for i in range(5)]
    plain, other = (beam.BeamSearch(2, 3, 4001, 5, end_ids=(7,)) for _ in range(2))
    caches = [torch.arange(6, dtype=torch.int32, device="cuda")[:, None].repeat(1, 9) for _ in range(2)]
    wanted = [plain.step(x, states=[caches[0]]).cpu() for x in steps]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy = torch.cuda.Event()
    torch.cuda._sleep(2_000_000_000)  # about a second
    busy.record()
    got = [other.step(x, states=[caches[1]], stream=side) for x in steps]
    side.synchronize()
    assert not busy.query()
    with torch.cuda.stream(side):
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, wanted))
    torch.cuda.synchronize()
    assert torch.equal(caches[0], caches[1]) and torch.equal(plain.tokens, other.tokens)
    assert torch.equal(plain.scores, other.scores) and torch.equal(plain.done, other.done)
    assert plain.best() == other.best()


def test_a_search_refuses_to_be_captured():
    torch = _torch()
    x = [_logits(6, 900, "f32", 60 + i) for i in range(3)]
    plain, run = (_beam().BeamSearch(2, 3, 900, 3) for _ in range(2))
    run.step(x[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x[1] + 1.0
        with pytest.raises(ValueError, match="captured"):
            run.step(x[1])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, x[1] + 1.0)
    run.step(x[1])
    run.step(x[2])
    for v in x:
        plain.step(v)
    assert torch.equal(run.tokens, plain.tokens) and torch.equal(run.scores, plain.scores)


def test_an_object_dropped_while_another_stream_works():
    # Its workspace and state are not handed out again before the stream that uses them is done.
    torch = _torch()
    beam = _beam()
    side = torch.cuda.Stream()
    x, s = _logits(6, 5000, "f32", 7), torch.from_numpy(_scores(2, 3, 1)).cuda()
    want = beam.BeamSelect(5000, 2, 3, 4)(x, s, 4)
    run = beam.BeamSearch(2, 3, 5000, 64)
    wanted = run.step(x).cpu()
    del run
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)  # about half a second
    select, run = beam.BeamSelect(5000, 2, 3, 4), beam.BeamSearch(2, 3, 5000, 64)
    side.wait_stream(torch.cuda.current_stream())  # the search's first contents
    mine = [select.workspace, run.select.workspace, run.tokens, run.done, run.scores, run.status]
    sizes, at = [t.numel() * t.element_size() for t in mine], {t.data_ptr() for t in mine}
    del mine
    got = select(x, s, 4, stream=side)
    new = run.step(x, stream=side)
    del select, run
    others = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(3)]
    assert not side.query()
    assert not at & {t.data_ptr() for t in others}
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(new.cpu(), wanted)


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_written_over_the_ones_before(dtype):
    # The C entry's promise where as many are kept as there are beams.
    torch = _torch()
    lib = S.load_library()
    x, s = _logits(40 * 5, 3001, dtype, 12), torch.from_numpy(_scores(40, 5, 3)).cuda()
    sel = _beam().BeamSelect(3001, 40, 5, 5)
    want = sel(x, s, 5)
    held = s.clone()
    tokens, parents = (torch.empty((40, 5), dtype=torch.int32, device="cuda") for _ in range(2))
    code = {"f32": S.TABBY_F32, "f16": S.TABBY_F16, "bf16": S.TABBY_BF16}[dtype]
    rc = lib.tabby_beam_select_device(x.data_ptr(), code, x.stride(0), 40, 5, 3001, held.data_ptr(), None, None, 0, 5,
                                      tokens.data_ptr(), parents.data_ptr(), held.data_ptr(), None, sel.workspace.data_ptr(),
                                      sel.workspace_bytes, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(held, want.scores) and torch.equal(tokens, want.tokens) and torch.equal(parents, want.parents)
