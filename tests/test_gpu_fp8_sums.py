"""The FP8 product's sums: held in f32 however many rows there are and whatever the result's type, unless fast ones are asked
for; and scales of any value."""
import numpy as np
import pytest

import fp8_oracle as F
import test_gpu_fp8 as P
from tabby_amd import sampler as S

pytestmark = pytest.mark.gpu

# Rows by weights' rows of every kernel: quantised in the launch, one to four tiles of rows, several groups of 64, tiles of 128 x 128
# in two groups of waves and in one, or of 256 x 256.
SIZES = [(1, 700), (9, 700), (30, 700), (45, 700), (64, 700), (65, 700), (260, 700), (300, 6001), (1000, 12501)]


def _codes(values):
    """The codes of float64 values that e4m3 holds."""
    codes = (F.nearest(np.abs(values)) | (np.signbit(values).astype(np.int64) << 7)).astype(np.uint8)
    assert np.array_equal(F.decoded(codes), values)
    return codes


def _held(values, scales):
    torch = P._torch()
    return P._fp8().Fp8Matrix.from_rowmajor(torch.from_numpy(_codes(values)).cuda(), torch.from_numpy(scales.astype(np.float32)).cuda())


@pytest.mark.parametrize("out", P.TYPES)
@pytest.mark.parametrize("rows,n", SIZES)
def test_what_is_left_where_large_products_cancel(rows, n, out):
    # In every eight columns two products of 448 x 448 that cancel, and six of whole numbers up to 2, in blocks whose scale is
    # one: all sums are whole numbers below 2^24, and what is left, up to some hundreds at k = 384, f16 holds exactly.
    torch = P._torch()
    k = 384
    rng = np.random.default_rng(rows + n)
    x, w = rng.integers(-1, 2, (rows, k)).astype(np.float64), rng.integers(-1, 2, (n, k)).astype(np.float64)
    x[:, 0::8] = x[:, 5::8] = 448.0
    w[:, 0::8], w[:, 5::8] = 448.0, -448.0
    m = _held(w, np.ones((-(-n // 128), 3)))
    want = x @ w.T
    assert np.abs(want).max() < 256  # whole numbers that bf16 holds too
    print(f"cancelling products {rows} x {n} to {out}", flush=True)
    got = P._fp8().matmul(torch.from_numpy(x).float().cuda(), m, dtype=P._dtype(out)).double().cpu().numpy()
    assert np.array_equal(got, want), np.abs(got - want).max()


FAST = [("f16", 70, 700), ("f16", 260, 700), ("f16", 300, 6001), ("f16", 1000, 6001), ("f16", 1000, 12501), ("bf16", 70, 700),
        ("bf16", 513, 5100), ("bf16", 300, 6001), ("bf16", 900, 6200), ("bf16", 1000, 12501)]


@pytest.mark.parametrize("out,rows,n", FAST)
def test_fast_sums_of_like_products_are_exact(out, rows, n):
    # Whole numbers up to 2: products of one sign or the other within 2^3 of each other, and sums that the result's type holds.
    # One dropped, doubled or changed for another shows.
    torch = P._torch()
    for k in (384, 130):
        rng = np.random.default_rng(rows + k)
        x, w = rng.integers(-2, 3, (rows, k)).astype(np.float64), rng.integers(-1, 3, (n, k)).astype(np.float64)
        x[:, 1::2] = -x[:, ::2]  # so that the weights' mean does not add up
        want = x @ w.T
        assert np.abs(want).max() <= 256
        m = _held(w, np.ones((-(-n // 128), -(-k // 128))))
        got = P._fp8().matmul(torch.from_numpy(x).float().cuda(), m, dtype=P._dtype(out), fast_sums=True).double().cpu().numpy()
        assert np.array_equal(got, want), np.argwhere(got != want)[:4]


@pytest.mark.parametrize("out,rows,n", FAST)
def test_fast_sums_take_each_block_with_its_own_scale(out, rows, n):
    # One block of each row of x nonzero, with a power of its own, and a power of its own to every block of the weights: the
    # sums are up to 144 times the smallest product.
    torch = P._torch()
    k = 1200
    rng = np.random.default_rng(2)
    x = np.zeros((rows, k))
    for r in range(rows):
        b = r % 10
        x[r, 128 * b:128 * b + 12] = rng.choice([-1.0, 1.0, 2.0, 3.0], 12) * 2.0 ** (r % 7)
    w = rng.choice([1.0, 0.5, 1.5, 2.0], (n, k))
    scales = np.exp2(rng.integers(-8, 1, (-(-n // 128), 10)))
    wv = w * scales.repeat(128, 0)[:n].repeat(128, 1)[:, :k]
    got = P._fp8().matmul(torch.from_numpy(x).float().cuda(), _held(w, scales), dtype=P._dtype(out), fast_sums=True).double().cpu().numpy()
    assert np.array_equal(got, x @ wv.T)


@pytest.mark.parametrize("out,rows,n", FAST)
def test_fast_sums_stay_within_their_bound(out, rows, n):
    # f32's sums, and seven of eight products to 2^-13 of the largest (test_gpu_fp8's bound); NaN reaches its row alone.
    torch = P._torch()
    x, exact = P._values(rows, 520, "bf16", rows + n, spread=0.3)
    w, wv = P._weights(n, 520, n)
    xv = F.rounded(exact)
    want = xv @ wv.T
    limit = P._bound(xv, wv, want, 520, out)
    got = P._fp8().matmul(x, w, dtype=P._dtype(out), fast_sums=True)
    again = P._fp8().matmul(P._fp8().Fp8Matrix.quantize(x), w, out=torch.empty_like(got), fast_sums=True)
    assert torch.equal(got, again)
    got = got.double().cpu().numpy()
    past = np.abs(want) > 65000 if out == "f16" else np.zeros(want.shape, dtype=bool)
    assert (np.abs(got - want) <= limit)[~past].all()
    x[rows // 2, 300] = float("nan")
    got = P._fp8().matmul(x, w, dtype=P._dtype(out), fast_sums=True)
    assert torch.isnan(got).all(1).nonzero().view(-1).tolist() == [rows // 2] and int(torch.isnan(got).sum()) == n


def test_fast_sums_where_they_make_no_difference_and_where_they_are_refused():
    torch = P._torch()
    x, _ = P._values(64, 520, "f16", 1)
    w, _ = P._weights(700, 520, 2, powers=True)
    for rows in (1, 16, 40, 64):
        for out in ("f16", "bf16"):
            a, b = (P._fp8().matmul(x[:rows], w, dtype=P._dtype(out), fast_sums=fast) for fast in (False, True))
            assert torch.equal(a, b)
    head = P._fp8().LmHeadFp8(w)
    assert torch.equal(head.logits(x, dtype=torch.bfloat16, fast_sums=True), P._fp8().matmul(x, w, dtype=torch.bfloat16, fast_sums=True))
    with pytest.raises(S.SamplingError, match="f16 and bf16 results"):
        P._fp8().matmul(x, w, fast_sums=True)
    with pytest.raises(S.SamplingError, match="f16 and bf16 results"):
        P._fp8().matmul(P._fp8().Fp8Matrix.quantize(x), w, out=torch.empty(64, 700, device="cuda"), fast_sums=True)


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", SIZES)
def test_scales_whose_product_is_no_f32(rows, n, out):
    # Both sides' scales lie within f32, their product above its largest value or below its smallest one, the result within
    # it: a block whose codes' sum is zero or small enough; or all of it among the smallest, with ordinary blocks beside.
    torch = P._torch()
    k = 640
    rng = np.random.default_rng(rows + n)
    x = np.zeros((rows, k))
    w = np.zeros((n, k))
    # Block 0: 2^110 times 2^25 and nothing that meets; block 1: the smallest codes, 2^-18 of 2^(110 + 20).
    x[:, 0], w[:, 1] = 448.0 * 2.0 ** 110, 448.0
    x[:, 128], x[:, 129], w[:, 129] = 448.0 * 2.0 ** 110, 2.0 ** -9 * 2.0 ** 110, 2.0 ** -9
    # Block 2: 2^-126 times 2^-20 or so of 3 x 448^2; block 3 as ordinary as can be; block 4 ordinary but for one row.
    x[:, 256:259], w[:, 256:259] = 448.0 * 2.0 ** -126, 448.0
    x[:, 384:400], w[:, 384:400] = rng.integers(-16, 17, (rows, 16)), rng.integers(-16, 17, (n, 16))
    x[:, 512:520], w[:, 512:520] = rng.integers(-16, 17, (rows, 8)), rng.integers(-16, 17, (n, 8))
    x[rows // 2, 512:520] *= 2.0 ** -100
    blocks = -(-n // 128)
    scales = np.ones((blocks, 5))
    scales[:, 0], scales[:, 1], scales[:, 2] = 2.0 ** 25, 2.0 ** 20, 1.37 * 2.0 ** -20
    scales[:, 3], scales[:, 4] = 0.9 * 2.0 ** -10, 0.7 * 2.0 ** -14

    def check(xs, ws, ss):
        m = _held(ws, ss)
        xv = F.rounded(xs.astype(np.float32))
        wv = ws * ss.astype(np.float32).astype(np.float64).repeat(128, 0)[:n].repeat(128, 1)[:, :k]
        want = xv @ wv.T
        # To f32's sums, and among the smallest values half a step to each block and one to the result.
        limit = P._bound(xv, wv, want, k, "f32") + 6 * 2.0 ** -150
        if out == "bf16":
            limit = limit + 2.0 ** -8 * (np.abs(want) + limit) + 2.0 ** -134
        got = P._fp8().matmul(torch.from_numpy(xs).float().cuda(), m, dtype=P._dtype(out)).double().cpu().numpy()
        assert np.isfinite(want).all() and (np.abs(got - want) <= limit).all(), np.argwhere(~(np.abs(got - want) <= limit))[:4]

    print(f"far scales {rows} x {n} to {out}", flush=True)
    check(x, w, scales)
    low, few = x.copy(), w.copy()
    low[:, :256] = 0.0
    low[:, 384:] = 0.0
    check(low, few, scales)  # only what lies among the smallest
    some = x.copy()
    some[: rows // 2, :384] = 0.0
    check(some, w, scales)   # rows of ordinary scales beside others
    scales[:, :3] = 0.0
    check(x, w, scales)      # weights' blocks that are empty
