"""Beam selection where the rows' sums decide: logits far from zero, fills of finite values, and beams whose
scores differ by less than f32 shows. Scores within f32's rounding of the sum in 64 bits."""
import numpy as np
import pytest

from test_gpu_beam import INF, TYPES, _beam, _dtype, _scores, _torch, choose

pytestmark = pytest.mark.gpu


def _select(x, scores, count, **more):
    torch = _torch()
    groups, beams = scores.shape
    sel = _beam().BeamSelect(vocab_max=x.shape[1], groups_max=groups, beams_max=beams, count_max=count)
    status = torch.full((groups,), -5, dtype=torch.int32, device="cuda")
    return sel(x, torch.from_numpy(scores).cuda(), count, status=status, **more), status


def _check(x, scores, count, ctx, copies=1):
    """`copies` of the groups in one call: many rows are not cut into parts, and a wave takes several chunks of one."""
    print(f"select {tuple(x.shape)} x {copies} keep {count} {x.dtype} {ctx}", flush=True)
    got, status = _select(x.repeat(copies, 1), np.tile(scores, (copies, 1)), count)
    exact = x.double().cpu().numpy()
    tokens, parents, best, states = (np.concatenate([a] * copies) for a in choose(exact, scores, count))
    assert np.array_equal(status.cpu().numpy(), states), ctx
    have = got.scores.double().cpu().numpy()
    assert not np.isnan(have).any(), ctx
    assert np.array_equal(got.tokens.cpu().numpy(), tokens), ctx
    assert np.array_equal(got.parents.cpu().numpy(), parents), ctx
    real = best > -INF
    assert np.array_equal(have > -INF, real), ctx
    # A term of the sum is off by 5.5e-11 of itself at most, the rest of the sum by some hundred steps of 2^-53,
    # and a score is three operations on numbers no larger than these; then f32 rounds once.
    finite = np.abs(exact[np.isfinite(exact)]).max()
    limit = 2.0 ** -24 * np.abs(best) + 1e-10 + 2.0 ** -50 * (np.abs(scores[np.isfinite(scores)]).max() + 2 * finite)
    err = np.abs(have[real] - best[real])
    assert (err <= limit[real]).all(), (ctx, err.max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [-680.0, -691.0, -710.0, -710.25, -2130.0, -7808.0, -58912.0])
def test_constant_rows_far_below_zero(value, dtype):
    torch = _torch()
    for groups, vocab in ((2, 700), (3, 9000), (1, 151936), (70, 20011)):
        x = torch.full((groups * 2, vocab), value, dtype=_dtype(dtype), device="cuda")
        _check(x, _scores(groups, 2, vocab), 5, f"all {value}")


def test_rows_about_the_end_of_the_doubles_range():
    # exp(-x) passes the largest number of 64 bits at x = -709.78.
    torch = _torch()
    rng = np.random.default_rng(710)
    for low, high in ((-711.0, -709.0), (-2131.0, -2128.0), (-745.5, -689.5)):
        x = torch.from_numpy(rng.uniform(low, high, (24, 12001)).astype(np.float32)).cuda()
        _check(x, _scores(6, 4, 1), 7, f"{low}..{high}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fill", [-710.0, -2130.0, -7808.0, -58912.0])
def test_stretches_of_a_finite_fill(fill, dtype):
    # A wave that meets nothing but the fill in its first chunk, and ordinary logits after it.
    torch = _torch()
    for vocab in (16384, 50257, 151936):
        rng = np.random.default_rng(vocab)
        x = rng.normal(0, 2.5, (8, vocab))
        x[0, :1024] = fill                       # the first wave's first chunk
        x[1, 3 * 1024:4 * 1024] = fill           # another's
        x[2, :vocab // 2] = fill                 # half a vocabulary
        x[3, :-1] = fill                         # all but the last entry
        x[4, 700:] = fill
        x[5, rng.random(vocab) < 0.999] = fill   # a mask that leaves little
        x[6] = fill
        for copies in (1, 33):
            _check(torch.from_numpy(x).to(_dtype(dtype)).cuda(), _scores(4, 2, vocab), 9, f"fill {fill}", copies)


@pytest.mark.parametrize("vocab", [5000, 40000])
def test_steps_that_f32_shows_coarsely(vocab):
    # Between 2^33 and 2^34 neighbouring logits are 1,024 apart, above it more; between 2^30 and 2^33 less.
    torch = _torch()
    for base in (2.0 ** 31, 2.0 ** 32, 2.0 ** 33, 2.0 ** 34, 2.0 ** 60, -2.0 ** 33, -2.0 ** 34, -2.0 ** 60):
        step = abs(base) * 2.0 ** -23
        x = np.full((6, vocab), base)
        for r, at in enumerate((0, 1023, 1024, vocab // 2, vocab - 1)):
            x[r, at] += step if base > 0 else step / 2
        x[5] += step * (np.arange(vocab) % 4)
        x = x.astype(np.float32)
        scores = np.array([[-1.0], [-2.0], [-3.0], [-4.0], [-5.0], [-6.0]], dtype=np.float32)
        for copies in (1, 44):
            _check(torch.from_numpy(x).cuda(), scores, 3, f"about {base}", copies)


@pytest.mark.parametrize("gap", [1e-8, 1e-9])
@pytest.mark.parametrize("vocab", [3001, 50257])
def test_the_order_of_beams_hangs_on_sums_in_64_bits(vocab, gap):
    # Two beams at one score with the same logits in another order, but for one entry that makes one row's sum larger
    # by `gap` of it: of every pair of equal logits the other beam's comes first. f32 sums are off by 1e-7.
    torch = _torch()
    rng = np.random.default_rng(vocab)
    groups = 60
    rows = np.empty((2 * groups, vocab), dtype=np.float32)
    for g in range(groups):
        a = rng.normal(0, 2.5, vocab).astype(np.float32)
        total = np.exp(a.astype(np.float64)).sum()
        b = a.copy()
        at = int(np.abs(a - 1.0).argmin())
        b[at] = np.log(np.exp(float(a[at])) + gap * total)
        grown = np.exp(b.astype(np.float64)).sum() / total - 1.0
        assert gap / 2 < grown < 2 * gap
        b = b[rng.permutation(vocab)]
        rows[2 * g], rows[2 * g + 1] = (a, b) if g % 2 else (b, a)
    scores = np.full((groups, 2), -7.25, dtype=np.float32)
    got, _ = _select(torch.from_numpy(rows).cuda(), scores, 8)
    smaller = (np.arange(groups) + 1) % 2
    want = np.stack([smaller, 1 - smaller] * 4, axis=1)
    assert np.array_equal(got.parents.cpu().numpy(), want)
    assert np.array_equal(got.tokens.cpu().numpy(), choose(rows.astype(np.float64), scores, 8)[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups,beams,vocab,count", [(1, 4, 151936, 8), (17, 4, 50257, 8), (70, 8, 20000, 16), (2, 3, 131, 5)])
def test_scores_within_their_rounding(groups, beams, vocab, count, dtype):
    torch = _torch()
    x = np.random.default_rng(vocab).normal(0, 2.5, (groups * beams, vocab))
    _check(torch.from_numpy(x).to(_dtype(dtype)).cuda(), _scores(groups, beams, vocab), count, "ordinary")
