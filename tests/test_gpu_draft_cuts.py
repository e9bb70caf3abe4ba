"""The verification's cuts where they are easily wrong: pools brought together from every number of lists, the largest
vocabulary, equal entries under a mask, tails of entries far lighter than the largest, and rows that cannot be used."""
import numpy as np
import pytest

import draft_oracle as D
import test_gpu_draft as V
from tabby_amd import sampler as S

pytestmark = pytest.mark.gpu

INF = float("inf")
NAN = float("nan")
LAST = np.nextafter(1.0, 0.0)  # the largest uniform


def _pools_agree(x, y, tokens, uniforms, lasts, settings, ctx):
    """Requests of as many drafted tokens each, top_k up to 128: x [requests, n + 1, vocab] and y [requests, n, vocab] of f32
    values. The oracle has only what lies among some row's first 128 entries, which keeps the vocabulary's order."""
    torch = V._torch()
    requests, n, vocab = y.shape
    print(f"pools {ctx}: {requests} requests of {n} x {vocab}", flush=True)
    v = V._draft().DraftVerify(vocab_max=vocab, requests_max=requests, drafts_max=n)
    status = torch.full((requests,), -5, dtype=torch.int32, device="cuda")
    got = v(x.view(-1, vocab), torch.from_numpy(tokens.reshape(-1).astype(np.int32)).cuda(), V._params(settings, lasts),
            torch.from_numpy(uniforms.reshape(-1)).cuda(), draft_logits=y.view(-1, vocab), status=status)
    assert status.tolist() == [0] * requests
    out, accepted = got.tokens.tolist(), got.accepted.tolist()
    # Of equal entries the lower index comes first: a stable sort.
    first = [torch.sort(t, dim=-1, descending=True, stable=True).indices[..., :128].cpu().numpy() for t in (x, y)]
    for r in range(requests):
        ids = np.unique(np.concatenate([f[r].ravel() for f in first] + [tokens[r]]))
        at = torch.from_numpy(ids).cuda()
        want, taken = D.decide(x[r][:, at].double().cpu().numpy(), np.searchsorted(ids, tokens[r]), uniforms[r], lasts[r], settings[r],
                               y[r][:, at].double().cpu().numpy())
        want = [int(ids[i]) for i in want]
        assert accepted[r] == taken and out[r] == want + [-1] * (n + 1 - len(want)), (ctx, r, settings[r], out[r], want)


def _rows_with_a_tail(shape, vocab, seed):
    """Rows whose largest entries lie among the last twentieth of the vocabulary, in part, and anywhere."""
    torch = V._torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, vocab, device="cuda", generator=g)
    last = vocab // 20
    x[..., -last:] += 6.0 * (torch.rand(*shape, last, device="cuda", generator=g) < 100.0 / last)
    return x + 5.0 * (torch.rand(*shape, vocab, device="cuda", generator=g) < 100.0 / vocab)


@pytest.mark.parametrize("vocab", [32768, 49152, 65536, 100352, 114688, 131072, 151936, 201088, 256000])
def test_pools_of_every_size_over_every_number_of_lists(vocab):
    # A row is cut into a list for each 16,384 entries, with so few rows: two to sixteen, brought together 64 entries at a
    # time, whatever the pool's size leaves of the last 64. The entries that matter lie in the last list.
    rng = np.random.default_rng(vocab)
    lists = -(-vocab // 16384)
    each = 512 // (3 * lists)  # requests of three rows, before rows are cut into fewer
    for first in range(1, 129, each):
        ks = list(range(first, min(first + each, 129)))
        x = _rows_with_a_tail((len(ks), 2), vocab, vocab + first)
        y = x[:, :1] + 0.3 * _rows_with_a_tail((len(ks), 1), vocab, vocab + first + 1)
        tokens = y.argmax(2).cpu().numpy()
        settings = [(1.0, k, 1.0 if k % 3 else 0.9) for k in ks]
        _pools_agree(x, y, tokens, rng.random((len(ks), 1)), rng.random(len(ks)), settings, f"top_k {ks[0]} to {ks[-1]}")


@pytest.mark.parametrize("top_k", [20, 50])
@pytest.mark.parametrize("requests,vocab", [(1, 151936), (6, 151936), (8, 151936), (1, 200064)])
def test_usual_pools_over_usual_vocabularies(requests, vocab, top_k):
    rng = np.random.default_rng(top_k)
    for seed in range(6):
        x = _rows_with_a_tail((requests, 5), vocab, seed)
        y = x[:, :4] + 0.2 * _rows_with_a_tail((requests, 4), vocab, seed + 100)
        tokens = y.argmax(2).cpu().numpy()
        _pools_agree(x, y, tokens, rng.random((requests, 4)), rng.random(requests), [(0.8, top_k, 0.95)] * requests, f"seed {seed}")


def _plain(x, settings, lasts):
    """The tokens drawn from rows without drafted ones."""
    torch = V._torch()
    none = torch.zeros(0, device="cuda")
    v = V._draft().DraftVerify(vocab_max=x.shape[1], requests_max=x.shape[0], drafts_max=0)
    status = torch.full((x.shape[0],), -5, dtype=torch.int32, device="cuda")
    got = v(x, none.int(), V._params(settings, lasts), none.double(), status=status, flags=S.TABBY_FLAG_FULL_VOCAB)
    assert status.tolist() == [0] * x.shape[0]
    return got.tokens[:, 0].tolist()


def test_a_number_of_entries_that_is_the_largest_vocabulary():
    # 2^24 equal entries: all of them in one bin.
    torch = V._torch()
    vocab = 2 ** 24
    settings = [(1.0, 200, 1.0), (0.5, 1000, 0.5), (1.0, 2 ** 24 - 1, 1.0), (2.0, 0, 0.25), (1e30, 4096, 1.0)]
    left = [200, 500, 2 ** 24 - 1, 2 ** 22, 4096]
    x = torch.full((1, vocab), 1.5, dtype=torch.bfloat16, device="cuda")
    for setting, n in zip(settings, left):
        print(f"largest vocabulary {setting}", flush=True)
        assert _plain(x, [setting], [0.0]) == [0]
        assert _plain(x, [setting], [LAST]) == [n - 1]
    # The same among several lists with some entries that are left out.
    x[:, ::2] = -INF
    assert _plain(x, [(1.0, 300, 1.0)], [LAST]) == [599]


@pytest.mark.parametrize("dtype", V.TYPES)
@pytest.mark.parametrize("setting", [(1.0, 0, 0.9), (0.8, 600, 0.95), (0.5, 2000, 1.0)])
def test_entries_that_no_bin_holds_beside_a_nan(setting, dtype):
    # A row's largest entries lie far above its reference and share 16 elements with a NaN: the row is refused, and no other.
    torch = V._torch()
    rng = np.random.default_rng(4)
    vocab, requests = 8192, 8
    x = V._logits(rng, 2 * requests, vocab)
    at = 64 * rng.integers(0, vocab // 64, requests) + 33
    far = 6e4 if dtype == "f16" else 1e30
    for r in range(0, requests, 2):
        for i, v in enumerate((40.0, 60.0, 75.0, far)):
            x[2 * r, (at[r] + 64 * i) % vocab] = NAN
            x[2 * r, (at[r] + 64 * i + 1) % vocab] = v
    tokens = np.where(np.isnan(x[::2]), -INF, x[::2]).argmax(1)
    target = torch.from_numpy(x).to(V._dtype(dtype)).cuda()
    V._check(target, tokens, rng.random(requests), rng.random(requests), [setting], [1] * requests, uniform_rows=True, bad_ok=True)


@pytest.mark.parametrize("count,top_p", [(10, 0.9), (10, 0.5), (1000, 0.9), (64, 0.25), (96, 0.75), (500, 0.2)])
@pytest.mark.parametrize("floor", [-INF, -80.0])
def test_equal_entries_under_a_mask(count, top_p, floor):
    # The tokens that a mask leaves are equally likely, at any logit, and lie where the row is not sampled for its
    # reference: top_p of `count` of them are a whole number.
    torch = V._torch()
    vocab, rows = 8192, 64
    left = int((np.cumsum(np.ones(count)) < top_p * count).sum()) + 1
    ids = 32 * np.arange(256)[:, None] + np.array([4, 9, 15, 21, 30])
    ids = np.sort(np.random.default_rng(count).permutation(ids.ravel())[:count])
    x = np.full((rows, vocab), floor)
    x[:, ids] = np.linspace(0.03, 9.0, rows)[:, None]
    got = _plain(torch.from_numpy(x).float().cuda(), [(0.7, 0, top_p)], [LAST] * rows)
    assert got == [int(ids[left - 1])] * rows


@pytest.mark.parametrize("vocab,tail,top_p,dtype", [(151936, -31.5, 1 - 1e-9, "f32"),
                                                    (2 ** 24, -27.0, 1 - 1e-5, "bf16"), (2 ** 24, -31.0, 1 - 2e-7, "bf16")])
@pytest.mark.parametrize("top_k", [0, -1])
@pytest.mark.parametrize("sampled", [True, False])
def test_a_wide_tail_far_below_the_largest(vocab, tail, top_p, dtype, sampled, top_k):
    # One entry, and all others alike and so light that only their number makes them matter: the cut lies among them where
    # the running sum says, to what the sums may be off by: 2^-52 of the largest to an entry, 2.5e-10 of the total where
    # it comes from the row's bins, and twice an exponential's 5.5e-11.
    torch = V._torch()
    peak = 0 if sampled else vocab // 3 // 4096 * 4096 + 1111  # the row's reference, or far above it
    x = torch.full((1, vocab), tail, dtype=V._dtype(dtype), device="cuda")
    x[0, peak] = 0.0
    weight = float(np.exp(x[0, 5].double().item()))
    k = vocab + top_k if top_k else 0
    entries = (k or vocab) - 1
    want = (top_p * (1 + entries * weight) - 1) / weight  # of the tail's entries; the index of the last, but for the peak's place
    off = (2.5e-10 + 1.2e-10 + vocab * 2.0 ** -52) / weight + 2
    assert 0.05 * vocab < off + want < 0.95 * vocab and off < 0.4 * vocab
    got = _plain(x, [(1.0, k, top_p)], [LAST])[0]
    assert abs(got - want) <= off, (got, want, off)


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("dtype", V.TYPES)
def test_rows_of_one_possible_token(dtype, with_draft):
    # All but one entry lie so far below it that they have no probability in 64 bits: a drafted token among them is refused, and
    # the one comes out, for uniforms of zero too, whichever of the others top_k left beside it.
    torch = V._torch()
    rng = np.random.default_rng(12)
    settings = [(0.05, 0, 1.0), (0.05, 0, 0.9), (0.05, 1102, 1.0), (0.05, 400, 0.99), (0.05, 40, 1.0), (0.05, 3000, 1.0)]
    vocab, requests = 3875, 12
    x = rng.normal(size=(2 * requests, vocab)) * 3
    y = x[::2] + rng.normal(size=(requests, vocab))
    for r in range(requests):
        peak = int(rng.integers(0, vocab))
        x[2 * r, peak] = y[r, peak] = 200.0
        x[2 * r + 1, rng.integers(0, vocab)] = 200.0
    target, draft = (torch.from_numpy(v).to(V._dtype(dtype)).cuda() for v in (x, y))
    for seed in range(4):
        rng = np.random.default_rng(seed)
        tokens = rng.integers(0, vocab, requests) if seed % 2 else x[::2].argmax(1)
        lasts = rng.random(requests) if seed < 2 else np.zeros(requests)
        V._check(target, tokens, rng.random(requests), lasts, settings, [1] * requests, draft if with_draft else None, uniform_rows=True)


@pytest.mark.parametrize("gap", [21.8, 22.0, 23.0])
def test_a_share_that_all_but_equals_top_p(gap):
    # Two equal entries, half of the total each but for a third one, the row's reference, of 1.7e-10 to 5e-11 of it: top_p 0.5
    # takes both.
    torch = V._torch()
    vocab, rows = 60000, 32
    x = np.full((rows, vocab), -300.0)
    rng = np.random.default_rng(3)
    want = []
    for r in range(rows):
        pair = 64 * np.sort(rng.permutation(vocab // 64 - 1)[:2]) + 37
        x[r, pair], x[r, 0] = 2.0 + r, 2.0 + r - gap
        share = np.nonzero(D.shares(x[r].astype(np.float32), 1.0, 0, 0.5))[0]
        assert share.tolist() == pair.tolist()
        want.append(int(pair[1]))
    got = _plain(torch.from_numpy(x).float().cuda(), [(1.0, 0, 0.5)], [LAST] * rows)
    assert got == want
