"""The verification of drafted tokens against its definition in 64 bits (draft_oracle): tokens and counts exactly."""
import ctypes

import numpy as np
import pytest

import draft_oracle as D
from tabby_amd import sampler as S

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16"]
INF = float("inf")
NAN = float("nan")
SETTINGS = {
    "pool": [(0.7, 40, 0.9)],
    "pools": [(0.7, 40, 0.9), (1.0, 1, 1.0), (1.3, 128, 1.0), (0.9, 33, 0.5), (0.01, 64, 0.99), (2.0, 5, 0.0)],
    "greedy": [(0.0, 0, 1.0), (-1.0, 7, 0.3)],
    "whole": [(1.0, 0, 1.0)],
    "nucleus": [(0.8, 0, 0.95), (1.5, 0, 0.5), (1.0, 0, 0.999)],
    "wide": [(1.0, 129, 0.98), (1.2, 1000, 1.0), (3.0, 400, 0.7)],
    "mixed": [(0.7, 40, 0.9), (1.0, 0, 1.0), (0.0, 1, 1.0), (0.8, 0, 0.95), (1.2, 100, 1.0), (1.0, 1000, 0.98)],
}


def _torch():
    import torch
    assert torch.cuda.is_available(), "needs an MI355X"
    return torch


def _draft():
    from tabby_amd import draft
    return draft


def _dtype(name):
    torch = _torch()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _params(settings, lasts):
    torch = _torch()
    p = np.zeros(len(lasts), dtype=S.PARAMS_DTYPE)
    for r, u in enumerate(lasts):
        t, k, top_p = settings[r % len(settings)]
        p[r] = (t, top_p, u, k, 0)
    return torch.from_numpy(p.view(np.uint8).copy()).cuda()


def _check(target, drafts, uniforms, lasts, settings, lengths, draft=None, uniform_rows=False, flags=S.TABBY_FLAG_FULL_VOCAB,
           verifier=None, ctx="", bad_ok=False):
    """`target` and `draft` CUDA tensors of packed rows; the rest numpy."""
    torch = _torch()
    requests, vocab = len(lengths), target.shape[1]
    most = max(lengths)
    at = np.cumsum([0] + [n + 1 for n in lengths])
    v = verifier or _draft().DraftVerify(vocab_max=vocab, requests_max=requests, drafts_max=most)
    print(f"verify {requests} requests {min(lengths)}..{most} drafts x {vocab} {target.dtype} draft={draft is not None} "
          f"{settings[:2]} {ctx}", flush=True)
    status = torch.full((requests,), -5, dtype=torch.int32, device="cuda")
    offsets = None if uniform_rows else torch.tensor(at, dtype=torch.int32, device="cuda")
    got = v(target, torch.from_numpy(drafts.astype(np.int32)).cuda(), _params(settings, lasts),
            torch.from_numpy(uniforms.astype(np.float64)).cuda(), draft_logits=draft, offsets=offsets, status=status, flags=flags)
    tokens, accepted, codes = got.tokens.cpu().numpy(), got.accepted.cpu().numpy(), status.cpu().numpy()
    x = target.double().cpu().numpy()
    y = None if draft is None else draft.double().cpu().numpy()
    for r, n in enumerate(lengths):
        d = at[r] - r
        want = D.decide(x[at[r]:at[r + 1]], drafts[d:d + n], uniforms[d:d + n], lasts[r], settings[r % len(settings)],
                        None if y is None else y[d:d + n])
        if want is None:
            assert bad_ok
            assert codes[r] == S.TABBY_EDOMAIN and accepted[r] == 0 and (tokens[r] == -1).all(), (r, codes[r], tokens[r])
            continue
        ids, taken = want
        assert codes[r] == S.TABBY_OK
        assert accepted[r] == taken, (r, accepted[r], taken, tokens[r], ids)
        assert tokens[r].tolist() == ids + [-1] * (tokens.shape[1] - len(ids)), (r, tokens[r], ids)
    return tokens, accepted


def _logits(rng, rows, vocab, hot=6, spread=2.0):
    x = rng.normal(size=(rows, vocab)) * spread
    for r in range(rows):
        x[r, rng.integers(0, vocab, hot)] = 7 + 4 * rng.random(hot)
    return x


def _case(requests, drafts, vocab, dtype, kind, with_draft, ragged, seed=0, noise=0.6):
    """Inputs whose drafted tokens are drawn from the draft, or mostly what the target says."""
    torch = _torch()
    rng = np.random.default_rng(seed + 1000 * requests + 17 * drafts + vocab)
    settings = SETTINGS[kind]
    lengths = [int(rng.integers(0, drafts + 1)) if ragged else drafts for _ in range(requests)]
    if ragged:
        lengths[0] = drafts
    rows, total = sum(lengths) + requests, sum(lengths)
    x = _logits(rng, rows, vocab)
    target = torch.from_numpy(x).to(_dtype(dtype)).cuda()
    before = [sum(lengths[:r]) + r + j for r in range(requests) for j in range(lengths[r])]
    draft = None
    if with_draft:
        draft = torch.from_numpy(x[before] + noise * rng.normal(size=(total, vocab))).to(_dtype(dtype)).cuda()
    source = (draft if with_draft else target[torch.tensor(before, dtype=torch.int64, device="cuda")]).double().cpu().numpy()
    owner = np.repeat(np.arange(requests), lengths)
    tokens = np.zeros(total, dtype=np.int64)
    for i in range(total):
        tokens[i] = D.drawn(D.shares(source[i], *settings[owner[i] % len(settings)]), rng.random())
        if not with_draft and rng.random() < 0.25:
            tokens[i] = rng.integers(0, vocab)
    return target, tokens, rng.random(total), rng.random(requests), settings, lengths, draft


@pytest.mark.parametrize("kind", sorted(SETTINGS))
@pytest.mark.parametrize("requests,drafts,vocab,dtype,with_draft,ragged", [
    (1, 4, 5000, "f32", True, False), (3, 2, 1000, "f16", True, True), (7, 5, 2049, "bf16", False, True),
    (2, 1, 129, "f32", True, False), (40, 3, 1500, "f32", True, True), (1, 8, 40001, "f16", False, False)])
def test_verified(kind, requests, drafts, vocab, dtype, with_draft, ragged):
    target, tokens, uniforms, lasts, settings, lengths, draft = _case(requests, drafts, vocab, dtype, kind, with_draft, ragged)
    _check(target, tokens, uniforms, lasts, settings, lengths, draft, uniform_rows=not ragged, ctx=kind)


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 64, 127, 128, 129, 130, 1023, 1025, 4095, 8193])
@pytest.mark.parametrize("kind", ["pools", "greedy", "whole", "nucleus", "wide"])
def test_small_vocabularies(vocab, kind):
    for dtype in TYPES:
        target, tokens, uniforms, lasts, settings, lengths, draft = _case(6, 3, vocab, dtype, kind, True, True)
        _check(target, tokens, uniforms, lasts, settings, lengths, draft, ctx=kind)


@pytest.mark.parametrize("kind", sorted(SETTINGS))
def test_nothing_drafted(kind):
    # No drafted token at all: plain sampling of one row to a request.
    torch = _torch()
    rng = np.random.default_rng(5)
    for requests in (1, 12):
        x = torch.from_numpy(_logits(rng, requests, 3001)).float().cuda()
        none = np.zeros(0)
        _check(x, none, none, rng.random(requests), SETTINGS[kind], [0] * requests, None, uniform_rows=True)
        _check(x, none, none, rng.random(requests), SETTINGS[kind], [0] * requests, None)


@pytest.mark.parametrize("kind", ["pool", "whole", "nucleus", "greedy"])
def test_large_vocabulary(kind):
    for requests, with_draft in ((1, True), (5, True), (70, False)):
        target, tokens, uniforms, lasts, settings, lengths, draft = _case(requests, 2, 151936, "f32", kind, with_draft, True)
        _check(target, tokens, uniforms, lasts, settings, lengths, draft, ctx=kind)


@pytest.mark.parametrize("kind", ["pools", "whole", "nucleus", "wide", "greedy"])
@pytest.mark.parametrize("dtype", TYPES)
def test_ties(kind, dtype):
    # Logits of few values, so that every cut falls among equal ones, and constant rows.
    torch = _torch()
    rng = np.random.default_rng(3)
    lengths, vocab = [2, 0, 3, 1, 2, 2], 3000
    rows, total = sum(lengths) + len(lengths), sum(lengths)
    x = np.round(rng.normal(size=(rows, vocab)) * 1.5)
    x[4] = 2.0
    x[7] = np.where(np.arange(vocab) % 2 == 0, 0.0, -0.0)
    y = np.round(rng.normal(size=(total, vocab)) * 1.5)
    y[3] = -1.0
    target, draft = (torch.from_numpy(v).to(_dtype(dtype)).cuda() for v in (x, y))
    for seed in range(4):
        rng = np.random.default_rng(seed)
        tokens = rng.integers(0, vocab, total)
        tokens[::2] = x[:total].argmax(1)[::2]
        _check(target, tokens, rng.random(total), rng.random(len(lengths)), SETTINGS[kind], lengths, draft if seed % 2 else None)


def test_equal_entries_are_cut_by_their_number():
    # 0.9 of 1,000 equal entries are 900 of them, the first 900; likewise where a pool was cut before.
    torch = _torch()
    for vocab, k, p, left in ((1000, 0, 0.9, 900), (1000, 0, 0.5, 500), (100, 0, 0.5, 50), (5000, 1000, 0.9, 900), (20000, 0, 0.25, 5000),
                              (300, 200, 0.5, 100), (64, 0, 0.25, 16), (20000, 10000, 0.5, 5000)):
        x = torch.zeros((2, vocab), device="cuda")
        v = _draft().DraftVerify(vocab_max=vocab, requests_max=2, drafts_max=0)
        top = np.nextafter(1.0, 0.0)
        none_i, none_f = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.float64, device="cuda")
        got = v(x, none_i, _params([(0.7, k, p)], [0.0, top]), none_f, flags=S.TABBY_FLAG_FULL_VOCAB)
        assert got.tokens[:, 0].tolist() == [0, left - 1], (vocab, k, p, got.tokens.tolist())


@pytest.mark.parametrize("kind", ["pools", "whole", "nucleus", "wide", "greedy", "mixed"])
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_rows(kind, dtype):
    # Rows masked down to some entries, to fewer than a pool has, and to one.
    torch = _torch()
    rng = np.random.default_rng(11)
    lengths, vocab = [3, 1, 2, 0, 3, 2], 6000
    rows, total = sum(lengths) + len(lengths), sum(lengths)
    x, y = _logits(rng, rows, vocab), _logits(rng, total, vocab)
    for v, keeps in ((x, (0.5, 20, 1, 0.1, 200)), (y, (0.3, 3, 50, 1))):
        for r in range(len(v)):
            keep = keeps[r % len(keeps)]
            left = rng.permutation(vocab)[: int(keep * vocab) if keep < 1 else keep]
            row = np.full(vocab, -INF)
            row[left] = v[r, left]
            v[r] = row
    target, draft = (torch.from_numpy(v).to(_dtype(dtype)).cuda() for v in (x, y))
    for seed in range(3):
        rng = np.random.default_rng(seed)
        tokens = np.array([rng.choice(np.nonzero(y[i] > -INF)[0]) for i in range(total)])
        _check(target, tokens, rng.random(total), rng.random(len(lengths)), SETTINGS[kind], lengths, draft if seed else None)


@pytest.mark.parametrize("order", ["ascending", "descending", "far", "peaks"])
@pytest.mark.parametrize("kind", ["pools", "nucleus", "wide", "whole"])
def test_unlikely_rows(order, kind):
    torch = _torch()
    rng = np.random.default_rng(2)
    rows, vocab = 6, 30000
    if order in ("ascending", "descending"):
        x = np.linspace(-9, 9, vocab)[None].repeat(rows, 0) + 0.01 * np.arange(rows)[:, None]
        if order == "descending":
            x = x[:, ::-1].copy()
    elif order == "far":  # logits further apart than exponentials reach
        x = rng.normal(size=(rows, vocab)) * 1e4
        x[1] = rng.choice([3e38, -3e38], vocab)
        x[2, 0], x[2, 1:] = 3.4e38, -3.4e38
    else:  # each chunk's maximum far above the last one's
        x = rng.normal(size=(rows, vocab)) + np.arange(vocab)[None] // 1024 * 700.0
    target = torch.from_numpy(x).float().cuda()
    draft = torch.from_numpy(x[[0, 1, 3, 4]] + 0.1 * rng.normal(size=(4, vocab))).float().cuda()
    tokens = x[[0, 1, 3, 4]].argmax(1)
    _check(target, tokens, rng.random(4), rng.random(2), SETTINGS[kind], [2, 2], draft)
    _check(target, tokens, rng.random(4), rng.random(2), SETTINGS[kind], [2, 2], None)


def test_temperatures_and_shares_at_the_edges():
    settings = [(1e-300, 0, 1.0), (5e-324, 0, 0.9), (1e308, 0, 0.5), (1e-3, 0, 0.9), (1e308, 50, 1.0), (1e-300, 50, 0.9), (1.0, 0, NAN),
                (1.0, 0, -3.0), (1.0, 0, 0.0), (1.0, 300, 1e-9), (1.0, 7, NAN), (1.0, 0, INF), (-INF, 5, 0.5), (1e30, 400, 0.9)]
    torch = _torch()
    for vocab in (700, 9000):
        rng = np.random.default_rng(vocab)
        n = len(settings)
        x = _logits(rng, 2 * n, vocab)
        target = torch.from_numpy(x).float().cuda()
        draft = torch.from_numpy(x[::2] + 0.3 * rng.normal(size=(n, vocab))).float().cuda()
        for given in (draft, None):
            tokens = x[::2].argmax(1)
            tokens[::3] = rng.integers(0, vocab, tokens[::3].size)
            _check(target, tokens, rng.random(n), rng.random(n), settings, [1] * n, given)


def test_uniforms_at_the_edges():
    # 0 accepts whatever has a probability at all, and draws the first token that has one.
    torch = _torch()
    rng = np.random.default_rng(8)
    vocab, top = 2000, np.nextafter(1.0, 0.0)
    x = _logits(rng, 8, vocab)
    target = torch.from_numpy(x).float().cuda()
    draft = torch.from_numpy(x[[0, 2, 4, 6]] + rng.normal(size=(4, vocab))).float().cuda()
    for kind in SETTINGS:
        for u in (0.0, top):
            for last in (0.0, top):
                for tokens in (x[[0, 2, 4, 6]].argmax(1), x[[0, 2, 4, 6]].argmin(1)):
                    for given in (draft, None):
                        _check(target, tokens, np.full(4, u), np.full(4, last), SETTINGS[kind], [1] * 4, given)


@pytest.mark.parametrize("kind", ["pool", "whole", "nucleus", "greedy"])
def test_the_same_distribution_accepts_everything(kind):
    torch = _torch()
    rng = np.random.default_rng(4)
    x = _logits(rng, 9, 5000)
    target = torch.from_numpy(x).float().cuda()
    draft = target[[0, 1, 3, 4, 6, 7]].contiguous()
    settings = SETTINGS[kind]
    tokens = np.array([D.drawn(D.shares(x[i].astype(np.float32), *settings[r % len(settings)]), rng.random())
                       for r in range(3) for i in (3 * r, 3 * r + 1)])
    _, accepted = _check(target, tokens, np.full(6, np.nextafter(1.0, 0.0)), rng.random(3), settings, [2] * 3, draft)
    assert accepted.tolist() == [2, 2, 2]


@pytest.mark.parametrize("setting", [(0.9, 5, 0.9), (1.0, 0, 1.0), (0.8, 0, 0.9)])
@pytest.mark.parametrize("certain", [False, True])
def test_tokens_are_distributed_as_the_targets(setting, certain):
    # One drafted token to each of many requests: the first token that comes out has the target's distribution.
    torch = _torch()
    rng = np.random.default_rng(77)
    vocab, requests = 200, 20000
    p_row, q_row = rng.normal(size=vocab) * 1.5, rng.normal(size=vocab) * 1.5
    q_row = (p_row + q_row) / 2
    target = torch.from_numpy(p_row).float().cuda()[None].expand(2 * requests, vocab).contiguous()
    draft = None if certain else torch.from_numpy(q_row).float().cuda()[None].expand(requests, vocab).contiguous()
    q = D.shares(q_row.astype(np.float32), *setting)
    tokens = np.full(requests, int(q.argmax())) if certain else rng.choice(vocab, size=requests, p=q)
    v = _draft().DraftVerify(vocab_max=vocab, requests_max=requests, drafts_max=1)
    got = v(target, torch.from_numpy(tokens.astype(np.int32)).cuda(), _params([setting], rng.random(requests)),
            torch.from_numpy(rng.random(requests)).cuda(), draft_logits=draft, flags=S.TABBY_FLAG_FULL_VOCAB)
    first = np.bincount(got.tokens[:, 0].cpu().numpy(), minlength=vocab) / requests
    p = D.shares(p_row.astype(np.float32), *setting)
    assert (first[p == 0] == 0).all()
    # Five standard deviations of each frequency.
    assert (np.abs(first - p) <= 5 * np.sqrt(p * (1 - p) / requests) + 1e-12).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows(dtype):
    torch = _torch()
    for kind in ("pools", "mixed"):
        target, tokens, uniforms, lasts, settings, lengths, draft = _case(5, 3, 2501, dtype, kind, True, True, seed=9)
        for lo, extra in ((0, 3), (1, 8), (5, 6)):
            wide = torch.full((target.shape[0], 2501 + extra + lo), 99.0, dtype=_dtype(dtype), device="cuda")
            wide[:, lo:lo + 2501] = target
            narrow = torch.full((draft.shape[0], 2501 + 1 + lo), 99.0, dtype=_dtype(dtype), device="cuda")
            narrow[:, lo:lo + 2501] = draft
            _check(wide[:, lo:lo + 2501], tokens, uniforms, lasts, settings, lengths, narrow[:, lo:lo + 2501])


def test_rows_that_cannot_be_used():
    # NaN, +inf and rows of -inf alone: only where they matter, and only their request.
    torch = _torch()
    rng = np.random.default_rng(21)
    vocab, lengths = 3000, [2] * 12
    for kind in ("pool", "whole", "nucleus", "greedy", "wide"):
        x = _logits(rng, 36, vocab)
        y = x[[3 * r + j for r in range(12) for j in range(2)]] + 0.05 * rng.normal(size=(24, vocab))
        x[0, 7], x[3 + 1, 9], x[6 + 2, 2999] = NAN, INF, NAN
        x[9 + 1], x[12, :] = -INF, -INF
        y[2 * 5, 3], y[2 * 6 + 1, 4], y[2 * 7] = NAN, INF, -INF
        x[24 + 2, 5] = NAN
        target, draft = torch.from_numpy(x).float().cuda(), torch.from_numpy(y).float().cuda()
        for u in (0.0, 0.999999):
            tokens = np.where(np.isnan(y), -INF, np.where(y == INF, -INF, y)).argmax(1)
            tokens[2 * 8 + 1] = int(x[24 + 1].argmin())
            for given in (draft, None):
                _check(target, tokens, np.full(24, u), rng.random(12), SETTINGS[kind], lengths, given, bad_ok=True, ctx=kind)


def test_requests_that_are_refused():
    torch = _torch()
    rng = np.random.default_rng(6)
    vocab = 1000
    x = torch.from_numpy(_logits(rng, 16, vocab)).float().cuda()
    v = _draft().DraftVerify(vocab_max=vocab, requests_max=8, drafts_max=1)
    good = (0.7, 40, 0.9)
    settings = [good, (NAN, 40, 0.9), (INF, 40, 0.9), (0.7, -1, 0.9), (0.7, 0, 0.9), (0.7, 129, 1.0), good, good]
    drafts = torch.zeros(8, dtype=torch.int32, device="cuda")
    drafts[6], drafts[7] = vocab, -1
    status = torch.full((8,), -5, dtype=torch.int32, device="cuda")
    uniforms = torch.zeros(8, dtype=torch.float64, device="cuda")
    got = v(x, drafts, _params(settings, [0.5] * 8), uniforms, status=status)
    assert status.tolist() == [S.TABBY_OK] + [S.TABBY_EINVAL] * 7
    assert (got.tokens[1:] == -1).all() and (got.accepted[1:] == 0).all() and int(got.tokens[0, 0]) >= 0
    got = v(x, drafts, _params(settings, [0.5] * 8), uniforms, status=status, flags=S.TABBY_FLAG_FULL_VOCAB)
    assert status.tolist() == [0, 1, 1, 1, 0, 0, 1, 1]
    reserved = _params([good], [0.5] * 8)
    reserved.view(torch.int32)[7] = 3
    got = v(x, torch.zeros_like(drafts), reserved, uniforms, status=status)
    assert status.tolist() == [1] + [0] * 7
    # A token outside the vocabulary after a refusal does not matter.
    w = _draft().DraftVerify(vocab_max=vocab, requests_max=1, drafts_max=2)
    got = w(x[:3], torch.tensor([int(x[0].argmin()), 5000], dtype=torch.int32, device="cuda"), _params([good], [0.5]),
            torch.full((2,), 0.5, dtype=torch.float64, device="cuda"), status=status[:1])
    assert status[:1].tolist() == [0] and got.accepted.tolist() == [0]


def test_offsets_outside_the_rows():
    # Requests whose rows, or whose drafted tokens (of 8: a row less for each request before), lie outside are refused,
    # each by itself; nothing is read outside.
    torch = _torch()
    rng = np.random.default_rng(6)
    vocab = 1000
    x = torch.from_numpy(_logits(rng, 12, vocab)).float().cuda()
    v = _draft().DraftVerify(vocab_max=vocab, requests_max=4, drafts_max=3)
    drafts = torch.from_numpy(rng.integers(0, vocab, 8).astype(np.int32)).cuda()
    uniforms = torch.full((8,), 0.5, dtype=torch.float64, device="cuda")
    status = torch.zeros(4, dtype=torch.int32, device="cuda")
    for offsets, want in (([0, 3, 6, 9, 12], [0, 0, 0, 0]), ([0, 4, 8, 12, 13], [0, 0, 1, 1]), ([0, 0, 4, 8, 12], [1, 1, 0, 0]),
                          ([-1, 3, 6, 9, 12], [1, 0, 0, 0]), ([0, 3, 2, 9, 12], [0, 1, 1, 0]), ([0, 1, 2, 3, 2 ** 31 - 1], [0, 0, 0, 1]),
                          ([-2 ** 31, 2 ** 31 - 1, 0, 4, 8], [1, 1, 1, 0]), ([9, 12, 12, 12, 12], [1, 1, 1, 1])):
        for flags in (0, S.TABBY_FLAG_FULL_VOCAB):
            v(x, drafts, _params([(0.7, 40, 0.9)] if not flags else [(0.7, 0, 0.9)], [0.5] * 4), uniforms, status=status, flags=flags,
              offsets=torch.tensor(offsets, dtype=torch.int64).to(torch.int32).cuda())
            assert status.tolist() == want, (offsets, status.tolist())


def test_an_object_serves_smaller_calls():
    verifier = _draft().DraftVerify(vocab_max=9000, requests_max=40, drafts_max=6)
    for seed, (requests, drafts, vocab, kind) in enumerate(((40, 6, 9000, "mixed"), (1, 6, 9000, "nucleus"), (3, 1, 50, "whole"),
                                                            (40, 0, 9000, "pool"), (2, 4, 8191, "wide"))):
        target, tokens, uniforms, lasts, settings, lengths, draft = _case(requests, drafts, vocab, "f32", kind, drafts > 0, False, seed=seed)
        _check(target, tokens, uniforms, lasts, settings, lengths, draft, uniform_rows=True, verifier=verifier)


def test_more_rows_than_units_and_many_drafts():
    target, tokens, uniforms, lasts, settings, lengths, draft = _case(90, 4, 2300, "f32", "mixed", True, True)
    _check(target, tokens, uniforms, lasts, settings, lengths, draft)
    target, tokens, uniforms, lasts, settings, lengths, draft = _case(3, 63, 700, "f32", "mixed", True, True, noise=0.02)
    _check(target, tokens, uniforms, lasts, settings, lengths, draft)


def test_nothing_is_written_outside():
    # The C entry with margins around its results and its workspace.
    torch = _torch()
    lib = S.load_library()
    target, tokens, uniforms, lasts, settings, lengths, draft = _case(9, 3, 5003, "f32", "mixed", True, False)
    size = ctypes.c_int64()
    assert lib.tabby_draft_workspace(9, 3, 5003, ctypes.byref(size)) == 0
    space = torch.full((size.value + 512,), 0xA5, dtype=torch.uint8, device="cuda")
    out = torch.full((36 + 9 + 9 + 40,), 1234, dtype=torch.int32, device="cuda")
    params = _params(settings, lasts)
    drafts, u = torch.from_numpy(tokens.astype(np.int32)).cuda(), torch.from_numpy(uniforms).cuda()
    at = out.data_ptr()
    rc = lib.tabby_draft_verify_device(
        target.data_ptr(), 0, 5003, 36, draft.data_ptr(), 5003, drafts.data_ptr(), u.data_ptr(), None, 9, 3, 5003, params.data_ptr(),
        at + 40, at + 40 + 36 * 4 + 40, at + 40 + 36 * 4 + 40 + 9 * 4 + 20, space.data_ptr() + 256, size.value, 1,
        torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.tabby_last_error()
    torch.cuda.synchronize()
    got = out.tolist()
    assert got[:10] == [1234] * 10 and got[46:56] == [1234] * 10 and got[65:70] == [1234] * 5 and got[79:] == [1234] * 15
    assert got[70:79] == [0] * 9
    assert (space[:256] == 0xA5).all() and (space[256 + size.value:] == 0xA5).all()
    v = _draft().DraftVerify(vocab_max=5003, requests_max=9, drafts_max=3)
    want = v(target, drafts, params, u, draft_logits=draft, flags=1)
    assert got[10:46] == want.tokens.view(-1).tolist() and got[56:65] == want.accepted.tolist()


def test_other_stream_and_graph():
    # On a stream of its own, and captured: every replay follows the inputs' present contents.
    torch = _torch()
    made = [_case(4, 3, 4000, "f32", "mixed", True, False, seed=s) for s in range(5)]
    v = _draft().DraftVerify(vocab_max=4000, requests_max=4, drafts_max=3)

    def dev(case):
        target, tokens, uniforms, lasts, settings, lengths, draft = case
        return [target, torch.from_numpy(tokens.astype(np.int32)).cuda(), _params(settings, lasts), torch.from_numpy(uniforms).cuda(), draft]
    side = torch.cuda.Stream()
    held = [t.clone() for t in dev(made[0])]
    torch.cuda.synchronize()
    got = v(*held[:4], draft_logits=held[4], flags=1, stream=side)
    side.synchronize()
    want = v(*held[:4], draft_logits=held[4], flags=1)
    assert torch.equal(got.tokens, want.tokens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = v(*held[:4], draft_logits=held[4], flags=1)
    for case in made:
        fresh = dev(case)
        for h, f in zip(held, fresh):
            h.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [out.tokens.clone(), out.accepted.clone()]
        want = v(*fresh[:4], draft_logits=fresh[4], flags=1)
        assert torch.equal(replayed[0], want.tokens) and torch.equal(replayed[1], want.accepted)
        torch.cuda.synchronize()


def test_host_form():
    torch = _torch()
    draft = _draft()
    rng = np.random.default_rng(3)
    vocab, lengths = 3000, [3, 0, 2, 1]
    settings = [S.SamplingParams(0.7, 40, 0.9), S.SamplingParams(0.0, 40, 0.9), S.SamplingParams(1.0, 0, 0.95), S.SamplingParams(0.9, 0, 1.0)]
    x = _logits(rng, 10, vocab)
    target = torch.from_numpy(x).float().cuda()
    drafts = [x[[0, 1, 2]].argmax(1).tolist(), [], x[[5, 6]].argmax(1).tolist(), [int(rng.integers(0, vocab))]]
    v = draft.DraftVerify(vocab_max=vocab, requests_max=4, drafts_max=3)
    got = v.verify(target, drafts, settings, S.SeededRandom(5))
    ref = S.SeededRandom(5)
    at = 0
    exact = target.double().cpu().numpy()
    for r, n in enumerate(lengths):
        s = settings[r]
        u = [ref.next() if s.temperature > 0 else 0.0 for _ in range(n)]
        last = ref.next() if s.temperature > 0 else 0.0
        ids, taken = D.decide(exact[at:at + n + 1], drafts[r], u, last, (s.temperature, s.topK, s.topP))
        assert got[r].tokens == ids and got[r].accepted == taken
        at += n + 1
    own = v.verify(target, drafts, settings, [S.SeededRandom(r) for r in range(4)])
    assert len(own) == 4
    with pytest.raises(S.SamplingError, match="request 1"):
        v.verify(target, drafts, [settings[0], S.SamplingParams(0.7, -2, 1.0), settings[2], settings[3]], S.SeededRandom(1))
    with pytest.raises(ValueError, match="temperature"):
        v.verify(target, drafts, S.SamplingParams(NAN, 5, 1.0), S.SeededRandom(1))
    with pytest.raises(ValueError, match="exceed the object"):
        v.verify(target, [[1] * 4, [], [], []], settings, S.SeededRandom(1))
    with pytest.raises(ValueError, match="random number generators"):
        v.verify(target, drafts, settings, [S.SeededRandom(1)])


def test_refusals():
    torch = _torch()
    draft = _draft()
    v = draft.DraftVerify(vocab_max=100, requests_max=2, drafts_max=2)
    x = torch.zeros(6, 100, device="cuda")
    d, u = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.float64, device="cuda")
    p = _params([(0.7, 5, 0.9)], [0.5, 0.5])
    v(x, d, p, u, draft_logits=x[:4])
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        v(x.double(), d, p, u)
    with pytest.raises(ValueError, match="evenly"):
        v(x[:5], d[:3], p, u[:3])
    with pytest.raises(ValueError, match="exceed the object"):
        v(torch.zeros(8, 100, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda"), p, torch.zeros(6, dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError, match="exceed the object"):
        v(torch.zeros(6, 101, device="cuda"), d, p, u)
    with pytest.raises(ValueError, match="drafts"):
        v(x, d[:3], p, u)
    with pytest.raises(ValueError, match="uniforms"):
        v(x, d, p, u.float())
    with pytest.raises(ValueError, match="draft_logits"):
        v(x, d, p, u, draft_logits=x[:4].half())
    with pytest.raises(ValueError, match="draft_logits"):
        v(x, d, p, u, draft_logits=x[:3])
    with pytest.raises(ValueError, match="params"):
        v(x, d, p[:33], u)
    with pytest.raises(ValueError, match="offsets"):
        v(x, d, p, u, offsets=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="status"):
        v(x, d, p, u, status=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(S.SamplingError, match="flags"):
        v(x, d, p, u, flags=2)
    with pytest.raises(S.SamplingError, match="overlap"):
        v(x, d, p, u, status=d[:2])
    with pytest.raises(S.SamplingError, match="between 0 and 63"):
        draft.DraftVerify(vocab_max=100, drafts_max=64)
    with pytest.raises(S.SamplingError, match="vocab"):
        draft.DraftVerify(vocab_max=2 ** 24 + 1)


def test_logits_past_32_bits():
    # 90,000 rows of 50,000 f32: the last requests' rows lie past 2^32 elements and 2^34 bytes.
    torch = _torch()
    rows, vocab, requests = 90_000, 50_000, 45_000
    x = torch.zeros((rows, vocab), device="cuda")
    x[:, 17] = 30.0
    x[rows - 2, 11], x[rows - 1, 49_999] = 60.0, 60.0
    v = _draft().DraftVerify(vocab_max=vocab, requests_max=requests, drafts_max=1)
    d = torch.full((requests,), 17, dtype=torch.int32, device="cuda")
    u = torch.full((requests,), 0.5, dtype=torch.float64, device="cuda")
    for setting, flags in (((0.7, 4, 1.0), 0), ((0.7, 0, 0.9), 1)):
        got = v(x, d, _params([setting], [0.5] * requests), u, flags=flags)
        assert got.accepted[:-1].min() == 1 and (got.tokens[:-1] == 17).all()
        assert got.accepted[-1] == 0 and got.tokens[-1].tolist() == [11, -1]
