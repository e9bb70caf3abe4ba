"""The FP8 heads and the verification of drafted tokens beyond their own files: cuts whose comparisons hang on the last bits,
batches without bins, windows that no list holds, calls side by side, and the operators together."""
import os
import sys

import numpy as np
import pytest

import draft_oracle as D
import fp8_oracle as F
import test_gpu_draft as V
import test_gpu_fp8 as P
from tabby_amd import sampler as S

pytestmark = pytest.mark.gpu


def _packed(case):
    """(target rows, draft rows or None, first row and number of drafted tokens of each request) as float64."""
    target, tokens, uniforms, lasts, settings, lengths, draft = case
    x = target.double().cpu().numpy()
    y = None if draft is None else draft.double().cpu().numpy()
    at = np.cumsum([0] + [n + 1 for n in lengths])
    return x, y, at


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["nucleus", "wide", "whole", "pools"])
@pytest.mark.parametrize("with_draft", [True, False])
def test_comparisons_that_hang_on_the_last_bits(kind, dtype, with_draft):
    # Every uniform is the ratio of the probabilities, a little more or a little less: by 1e-8, many times what
    # the probabilities may be off by (the exponentials' 5.5e-11, twice, of each), far less than bins of a sixteenth of an octave tell.
    for seed, off in enumerate((1e-8, 1e-6, 1e-3)):
        case = list(V._case(12, 5, 3001, dtype, kind, with_draft, True, seed=seed))
        x, y, at = _packed(case)
        rng = np.random.default_rng(seed)
        uniforms, settings, lengths = case[2], case[4], case[5]
        for r, n in enumerate(lengths):
            for j in range(n):
                i = at[r] - r + j
                s = settings[r % len(settings)]
                p = D.shares(x[at[r] + j], *s)[case[1][i]]
                q = D.shares(y[i], *s)[case[1][i]] if with_draft else 1.0
                # (One in four a plain refusal, or there would be none where all hold.)
                uniforms[i] = p / q * (1 + off * (1 if rng.random() < 0.25 else -1)) if q > 0 else rng.random()
                uniforms[i] = min(uniforms[i], 1 - 2.0 ** -53)
        tokens, accepted = V._check(*case, ctx=f"{kind} {off}")
    assert accepted.max() > 0


@pytest.mark.parametrize("requests,drafts,vocab", [(1500, 1, 300), (460, 4, 500), (5000, 0, 400)])
def test_more_rows_than_have_bins(requests, drafts, vocab):
    # More than 4,096 lists: whole vocabularies are cut without bins.
    case = V._case(requests, drafts, vocab, "f32", "mixed" if drafts else "wide", drafts > 0, False)
    V._check(*case, uniform_rows=True)


@pytest.mark.parametrize("dtype", V.TYPES)
def test_windows_that_no_list_holds(dtype):
    # Equal logits, all or all but a few: the cut lies among more entries than are gathered or held at once, at a number of
    # them that is exact.
    torch = V._torch()
    vocab, rng = 20011, np.random.default_rng(1)
    settings = [(1.0, 0, 0.9), (0.7, 7000, 1.0), (1.0, 9000, 0.5), (2.0, 0, 0.123)]
    x = np.zeros((12, vocab))
    x[3:6] = rng.integers(0, 2, (3, vocab))
    x[6:9, rng.integers(0, vocab, 40)] = 1.5
    x[9:] = np.where(np.arange(vocab) < 6000, 1.0, -3.0)
    target = torch.from_numpy(x).to(V._dtype(dtype)).cuda()
    draft = torch.from_numpy(np.roll(x, 5, axis=1)[[0, 1, 3, 4, 6, 7, 9, 10]]).to(V._dtype(dtype)).cuda()
    tokens = np.array([int(rng.integers(0, 3000)) for _ in range(8)])
    for seed in range(3):
        rng = np.random.default_rng(seed)
        V._check(target, tokens, rng.random(8), rng.random(4), settings, [2] * 4, draft, uniform_rows=True, ctx="equal")


@pytest.mark.parametrize("vocab", [30000, 151936])
def test_likely_tokens_side_by_side(vocab):
    # All that may be left lies at the beginning, at the end, or in one stretch: one share of the gathering has it all.
    torch = V._torch()
    rng = np.random.default_rng(2)
    settings = [(1.0, 0, 0.97), (0.8, 3000, 0.99)]
    for first in (0, vocab - 4000, 12345):
        x = rng.normal(size=(6, vocab)) * 0.5 - 20
        x[:, first:first + 4000] = rng.normal(size=(6, 4000))
        draft = torch.from_numpy(x[[0, 1, 3, 4]] + 0.1 * rng.normal(size=(4, vocab))).float().cuda()
        tokens = np.array([int(first + rng.integers(0, 4000)) for _ in range(4)])
        V._check(torch.from_numpy(x).float().cuda(), tokens, rng.random(4), rng.random(2), settings, [2, 2], draft, uniform_rows=True,
                 ctx=f"from {first}")


def test_logits_far_above_the_sample():
    # The bins lie relative to the largest of some loads spread over the row; one entry elsewhere far above it, or
    # temperatures that spread the row over more than they hold.
    torch = V._torch()
    vocab, rng = 70001, np.random.default_rng(3)
    settings = [(1.0, 0, 0.9), (1e-3, 0, 0.99), (0.5, 500, 0.9), (50.0, 0, 0.999)]
    x = rng.normal(size=(12, vocab)) * 2
    for r in range(12):
        x[r, rng.integers(0, vocab, 3)] = [40.0, 300.0, 300.5] if r % 3 else [23.0, 22.5, 22.0]
    draft = torch.from_numpy(x[[0, 1, 3, 4, 6, 7, 9, 10]] + 0.05 * rng.normal(size=(8, vocab))).float().cuda()
    tokens = x[[0, 1, 3, 4, 6, 7, 9, 10]].argmax(1)
    for seed in range(3):
        rng = np.random.default_rng(seed)
        V._check(torch.from_numpy(x).float().cuda(), tokens, rng.random(8), rng.random(4), settings, [2] * 4, draft, uniform_rows=True)


def test_objects_side_by_side():
    # Two objects on two streams at once, their launches in turn: each has its own results.
    torch = V._torch()
    made = [V._case(6, 4, 30011, "f32", kind, True, False, seed=s) for s, kind in enumerate(("nucleus", "mixed"))]
    inputs = []
    for target, tokens, uniforms, lasts, settings, lengths, draft in made:
        inputs.append([target, torch.from_numpy(tokens.astype(np.int32)).cuda(), V._params(settings, lasts),
                       torch.from_numpy(uniforms).cuda(), draft])
    objects = [V._draft().DraftVerify(vocab_max=30011, requests_max=6, drafts_max=4) for _ in made]
    want = [v(*i[:4], draft_logits=i[4], flags=1).tokens.clone() for v, i in zip(objects, inputs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    got = [[], []]
    for _ in range(10):
        for s, (v, i) in enumerate(zip(objects, inputs)):
            got[s].append(v(*i[:4], draft_logits=i[4], flags=1, stream=streams[s]).tokens)
    torch.cuda.synchronize()
    for s in range(2):
        assert all(torch.equal(g, want[s]) for g in got[s])


@pytest.mark.parametrize("dtype", P.TYPES)
@pytest.mark.parametrize("rows,k", [(1, 4096), (1, 4097), (16, 256), (16, 257), (17, 128), (10, 384), (11, 384), (2, 2048), (3, 2000), (5, 800)])
def test_rows_quantised_in_the_products_launch(rows, k, dtype):
    # Up to 16 rows and 32 of their blocks, on either side of both limits: the same to the last bit as quantised before.
    torch = P._torch()
    for n in (64, 1000, 20000):
        w, _ = P._weights(n, k, n + k)
        x, _ = P._values(rows, k, dtype, rows + k)
        print(f"fills {rows} x {n} x {k} {dtype}", flush=True)
        held = P._fp8().Fp8Matrix.quantize(x)
        for out in (torch.float32, torch.bfloat16):
            assert torch.equal(P._fp8().matmul(x, w, dtype=out), P._fp8().matmul(held, w, dtype=out))
    wide = torch.full((rows, k + 7), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, 3:3 + k] = x
    assert torch.equal(P._fp8().matmul(wide[:, 3:3 + k], w), P._fp8().matmul(held, w))


@pytest.mark.parametrize("k", [100, 300, 390])
@pytest.mark.parametrize("rows,n,out", [(300, 5600, "f16"), (300, 10800, "f32"), (513, 5100, "bf16")])
def test_product_in_two_groups(rows, n, k, out):
    # Between half as many tiles of 128 x 128 as units and one to each: k in two groups of waves, the second with a panel less or none.
    P._check_product(rows, n, k, P.TYPES[k % 3], out, k == 300)


def test_example_runs_the_heads_and_the_verification_together():
    # examples/speculative_fp8.py: its logits against the values that the heads stand for, its tokens against the definition.
    torch = V._torch()
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import speculative_fp8 as example
    vocab, hidden, drafts = 1003, 160, 3
    target = example.Model(vocab, hidden, seed=3)
    proposer = example.Model(vocab, hidden, seed=4, near=target, noise=0.5)
    settings = [S.SamplingParams(0.7, 40, 0.9), S.SamplingParams(1.0, 0, 0.95), S.SamplingParams(0.0, 1, 1.0), S.SamplingParams(1.3, 0, 1.0),
                S.SamplingParams(0.9, 500, 0.98)]
    run = example.Speculation(target, proposer, settings, drafts)
    tokens = torch.tensor([5, 77, 1002, 0, 400], dtype=torch.int32, device="cuda")
    weights = [m.head.weight.dequantize().double().cpu().numpy() for m in (target, proposer)]
    embed = target.embed.double().cpu().numpy()
    taken = 0
    for _ in range(4):
        step = run.step(tokens)
        x, y = step.logits.double().cpu().numpy(), step.draft_logits.double().cpu().numpy()
        d, u = step.drafts.cpu().numpy(), step.uniforms.cpu().numpy()
        ids, accepted = step.verified.tokens.tolist(), step.verified.accepted.tolist()
        for r, s in enumerate(settings):
            last = [int(tokens[r])] + d[r * drafts:(r + 1) * drafts].tolist()
            for got, w, of in ((x[r * (drafts + 1):(r + 1) * (drafts + 1)], weights[0], last), (y[r * drafts:(r + 1) * drafts], weights[1], last[:-1])):
                h = F.rounded(embed[of])
                want = h @ w.T
                assert (np.abs(got - want) <= P._bound(h, w, want, hidden, "f32")).all()
            want = D.decide(x[r * (drafts + 1):(r + 1) * (drafts + 1)], last[1:], u[r * drafts:(r + 1) * drafts], float(step.lasts[r]),
                            (s.temperature, s.topK, s.topP), y[r * drafts:(r + 1) * drafts])
            assert (ids[r][:accepted[r] + 1], accepted[r]) == (want[0], want[1])
            taken += accepted[r]
        tokens = torch.tensor([i[n] for i, n in zip(ids, accepted)], dtype=torch.int32, device="cuda")
    assert taken > 0
    made, steps = run.generate(tokens, 5)
    assert min(map(len, made)) >= 5 and 1 <= steps <= 5 and all(0 <= t < vocab for m in made for t in m)
