"""The MXFP4 operators against their definition in 64 bits (mx4_oracle): conversion and the way
back bit for bit, the product within its accumulation's bound, at odd sizes, strides and types,
and with blocks that hold zeros, subnormals, infinities and NaN."""
import numpy as np
import pytest

import mx4_oracle as M
from tabby_amd import sampler as S

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16"]


def _torch():
    import torch
    assert torch.cuda.is_available(), "needs an MI355X"
    return torch


def _dtype(name):
    torch = _torch()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _values(rows, cols, dtype, seed, spread=1.0):
    """(tensor of `dtype` on the GPU, its exact float64 values)."""
    torch = _torch()
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(rows, cols)) * np.exp(spread * rng.normal(size=(rows, cols)))
    t = torch.from_numpy(x).to(_dtype(dtype))
    return t.cuda(), t.double().numpy()


def _mx4():
    from tabby_amd import mx4
    return mx4


def _same(got, want):
    return np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (1, 32), (2, 33), (15, 127), (16, 128), (17, 129), (64, 896),
                                       (65, 1000), (130, 4850)])
def test_round_trip(rows, cols, dtype):
    x, exact = _values(rows, cols, dtype, rows * 10007 + cols)
    print(f"round trip {rows} x {cols} {dtype}", flush=True)
    m = _mx4().Mx4Matrix.quantize(x)
    want = M.rounded(exact)
    for back in TYPES:
        got = m.dequantize(_dtype(back)).double().cpu().numpy()
        assert got.shape == (rows, cols)
        held = _torch().from_numpy(want).to(_dtype(back)).double().numpy()
        assert _same(got, held), (back, np.argwhere(got != held)[:4])
        if back == "bf16":
            assert _same(got, want)  # a code times a power of two always fits


def test_every_code_and_every_tie():
    # A block led by 6 * 2^E has the power E: all sixteen codes, the seven midpoints of both signs, and
    # the neighbours of each midpoint in f32, over many powers.
    torch = _torch()
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    near = [v for m in mids for v in (np.nextafter(np.float32(m), np.float32(0)), m, np.nextafter(np.float32(m), np.float32(9)))]
    pool = np.array(list(M.LEVELS) + near + [7.9, 6.5, -0.0], dtype=np.float32)
    pool = np.concatenate([pool, -pool])
    rows = []
    for e in (-126, -120, -100, -24, -3, 0, 1, 17, 80, 125):
        for i in range(0, len(pool), 31):
            part = np.zeros(32, dtype=np.float32)
            part[0] = 6.0
            part[1:1 + len(pool[i:i + 31])] = pool[i:i + 31]
            rows.append(np.ldexp(part.astype(np.float64), e).astype(np.float32))
    x = np.stack(rows)
    m = _mx4().Mx4Matrix.quantize(torch.from_numpy(x).cuda())
    got = m.dequantize().cpu().numpy().astype(np.float64)
    want = M.rounded(x)
    assert _same(got, want), [(x[i, j], got[i, j], want[i, j]) for i, j in np.argwhere(got != want)[:6]]


def test_powers_at_both_ends():
    # The exponent is held to [-127, 127]: subnormals below 2^-127, f32's largest values above.
    torch = _torch()
    x = np.zeros((9, 64), dtype=np.float32)
    x[0, :4] = [1e-45, -1e-45, 0, 0]
    x[1, :4] = [2.0 ** -126, 2.0 ** -127, 2.0 ** -128, 2.0 ** -129]
    x[2, :4] = [3 * 2.0 ** -125, 2.0 ** -126, -(2.0 ** -127), 2.0 ** -149]
    x[3, :4] = [np.finfo(np.float32).max, 2.0 ** 127, -(2.0 ** 125), 1.0]
    x[4, 32:36] = [2.0 ** -124, 2.0 ** -125, 1.5 * 2.0 ** -126, 2.0 ** -127]
    x[5, 0], x[5, 40] = np.inf, 3.0
    x[6, 63], x[6, 1] = np.nan, 5.0
    x[7, 2], x[7, 3] = -np.inf, np.nan
    got = _mx4().Mx4Matrix.quantize(torch.from_numpy(x).cuda()).dequantize().cpu().numpy().astype(np.float64)
    want = M.rounded(x)
    assert _same(got, want), [(i, j, x[i, j], got[i, j], want[i, j]) for i, j in np.argwhere((got != want) & ~np.isnan(want))[:8]]
    assert np.isnan(got[5, :32]).all() and not np.isnan(got[5, 32:]).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_unaligned_rows(dtype):
    torch = _torch()
    base, exact = _values(40, 700, dtype, 5)
    for lo, cols in ((0, 640), (1, 333), (3, 64), (8, 257)):
        x = base[:, lo:lo + cols]
        got = _mx4().Mx4Matrix.quantize(x).dequantize(out=torch.full((40, 800), 7.0, device="cuda")[:, 5:5 + cols])
        assert _same(got.double().cpu().numpy(), M.rounded(exact[:, lo:lo + cols])), (lo, cols)
    odd = torch.full((40, 801), 7.0, device="cuda", dtype=_dtype(dtype))
    _mx4().Mx4Matrix.quantize(base[:, :640]).dequantize(out=odd[:, 80:720])
    want = torch.from_numpy(M.rounded(exact[:, :640])).to(_dtype(dtype)).double().numpy()
    assert _same(odd[:, 80:720].double().cpu().numpy(), want)
    assert (odd[:, :80] == 7.0).all() and (odd[:, 720:] == 7.0).all()  # nothing beside the rows is written


@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 31), (16, 32), (33, 100), (64, 128), (100, 896), (7, 1027)])
def test_checkpoint_layout(rows, cols):
    torch = _torch()
    rng = np.random.default_rng(rows + cols)
    blocks = -(-cols // 32)
    codes = rng.integers(0, 16, (rows, blocks * 32), dtype=np.uint8)
    scales = rng.integers(0, 255, (rows, blocks), dtype=np.uint8)
    scales[rng.random((rows, blocks)) < 0.05] = 255
    m = _mx4().Mx4Matrix.from_rowmajor(torch.from_numpy(M.packed(codes)).cuda(), torch.from_numpy(scales).cuda(), cols)
    with np.errstate(over="ignore"):
        want = M.values(codes, scales, cols).astype(np.float32)  # 2 * 2^127 and above: infinite in f32
    assert _same(m.dequantize().cpu().numpy(), want)


def test_buffers_are_written_again():
    torch = _torch()
    a, _ = _values(50, 200, "f32", 1)
    b, exact = _values(50, 200, "bf16", 2)
    m = _mx4().Mx4Matrix.quantize(a)
    assert _mx4().Mx4Matrix.quantize(b, out=m) is m
    assert _same(m.dequantize().cpu().numpy().astype(np.float64), M.rounded(exact))


def _weights(n, k, seed, low=118, high=124):
    """(Mx4Matrix, float64 values) of random codes."""
    torch = _torch()
    rng = np.random.default_rng(seed)
    blocks = -(-k // 32)
    codes = rng.integers(0, 16, (n, blocks * 32), dtype=np.uint8)
    scales = rng.integers(low, high, (n, blocks), dtype=np.uint8)
    m = _mx4().Mx4Matrix.from_rowmajor(torch.from_numpy(M.packed(codes)).cuda(), torch.from_numpy(scales).cuda(), k)
    return m, M.values(codes, scales, k)


def _bound(x, w, y, k, out, bias=None):
    """Accumulation in f32, at most one step of 2^-23 relative to an add (k of them and the bias's), then
    one rounding to the output's type."""
    torch = _torch()
    grown = np.abs(x) @ np.abs(w).T + (0 if bias is None else np.abs(bias))
    eps = torch.finfo(_dtype(out)).eps
    tiny = torch.finfo(_dtype(out)).smallest_normal
    return (k + 1) * 2.0 ** -23 * grown + eps / 2 * (np.abs(y) + k * 2.0 ** -23 * grown) + tiny * eps


def _check_product(rows, n, k, dtype, out, bias, seed=0):
    torch = _torch()
    x, exact = _values(rows, k, dtype, 31 * rows + n + seed, spread=0.3)
    w, wv = _weights(n, k, 7 * n + k + seed)
    b = np.random.default_rng(n).normal(size=n).astype(np.float32) if bias else None
    head = _mx4().LmHeadMx4(w, None if b is None else torch.from_numpy(b).cuda())
    print(f"product {rows} x {n} x {k} {dtype}->{out} bias={bias}", flush=True)
    xv = M.rounded(exact)
    want = xv @ wv.T + (0 if b is None else b.astype(np.float64))
    limit = _bound(xv, wv, want, k, out, b)
    got = head.logits(x, dtype=_dtype(out))
    assert got.shape == (rows, n) and got.dtype == _dtype(out)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= limit).all(), (err.max(), np.argwhere(err > limit)[:4])
    again = _mx4().matmul(_mx4().Mx4Matrix.quantize(x), w, head.bias, dtype=_dtype(out))
    assert torch.equal(got, again)  # quantised in the call or before it


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 64, 128), (1, 1000, 896), (2, 63, 31), (3, 65, 160), (15, 17, 33),
                                      (16, 200, 1024), (17, 129, 257), (31, 96, 64), (33, 300, 800), (64, 64, 4096),
                                      (65, 257, 640), (100, 1000, 1000), (128, 512, 384), (129, 255, 897), (257, 300, 513),
                                      (300, 1027, 896), (513, 520, 2056)])
def test_product(rows, n, k):
    i = rows + n + k
    _check_product(rows, n, k, TYPES[i % 3], TYPES[(i // 3) % 3], i % 2 == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("rows", [1, 24, 200])
def test_product_types(dtype, out, rows):
    _check_product(rows, 333, 416, dtype, out, rows != 24)


@pytest.mark.parametrize("rows", [1, 5, 16, 40, 70, 260])
def test_exact_sums(rows):
    # Codes with power 0: every sum is a multiple of 1/4 far below 2^24, so f32 holds it exactly,
    # whatever the order.
    torch = _torch()
    n, k = 700, 1500
    rng = np.random.default_rng(rows)
    codes = rng.integers(0, 16, (rows, 47 * 32), dtype=np.uint8)
    ones = np.full((rows, 47), 127, dtype=np.uint8)
    x = _mx4().Mx4Matrix.from_rowmajor(torch.from_numpy(M.packed(codes)).cuda(), torch.from_numpy(ones).cuda(), k)
    w, wv = _weights(n, k, 3, 127, 128)
    got = _mx4().matmul(x, w).cpu().numpy().astype(np.float64)
    assert np.array_equal(got, M.values(codes, ones, k) @ wv.T)


def test_each_block_has_its_own_scales():
    # One block of each side nonzero at a time, with powers of its own: a value or scale taken from
    # another block, row or tile shows.
    torch = _torch()
    rows, n, k = 70, 130, 300
    rng = np.random.default_rng(1)
    x, w = np.zeros((rows, k)), np.zeros((n, k))
    for r in range(rows):
        b = r % 10
        x[r, 32 * b:32 * b + 12] = rng.choice([-1.0, 1.0, 2.0, 3.0], 12) * 2.0 ** (r % 7)
    for c in range(n):
        b = (3 * c) % 10
        w[c, 32 * b:32 * b + 12] = rng.choice([1.0, -0.5, 1.5], 12) * 2.0 ** (-(c % 11))
    t = lambda a: _mx4().Mx4Matrix.quantize(torch.from_numpy(a).float().cuda())
    got = _mx4().matmul(t(x), t(w)).cpu().numpy().astype(np.float64)
    assert np.array_equal(got, M.rounded(x) @ M.rounded(w).T)


@pytest.mark.parametrize("rows", [2, 20, 90])
def test_nan_blocks_reach_their_rows_alone(rows):
    torch = _torch()
    x, exact = _values(rows, 200, "f32", 3)
    x[1, 190] = float("inf")
    w, wv = _weights(150, 200, 4)
    got = _mx4().matmul(x, w).cpu().numpy()
    assert np.isnan(got[1]).all()
    assert np.isfinite(np.delete(got, 1, 0)).all()
    wq = _mx4().Mx4Matrix.quantize(torch.from_numpy(np.where(np.arange(150)[:, None] == 149, np.nan, wv)).float().cuda())
    got = _mx4().matmul(x[2:] if rows > 2 else x[:1], wq).cpu().numpy()
    assert np.isnan(got[:, 149]).all() and np.isfinite(got[:, :149]).all()


@pytest.mark.parametrize("rows", [1, 30, 140])
def test_product_into_strided_output(rows):
    torch = _torch()
    x, exact = _values(rows, 320, "bf16", 9)
    w, wv = _weights(203, 320, 10)
    for out in TYPES:
        wide = torch.full((rows, 300), 5.0, device="cuda", dtype=_dtype(out))
        for lo in (0, 1, 4, 7):
            wide.fill_(5.0)
            _mx4().matmul(x, w, out=wide[:, lo:lo + 203])
            want = M.rounded(exact) @ wv.T
            err = np.abs(wide[:, lo:lo + 203].double().cpu().numpy() - want)
            assert (err <= _bound(M.rounded(exact), wv, want, 320, out)).all()
            assert (wide[:, :lo] == 5.0).all() and (wide[:, lo + 203:] == 5.0).all()


def test_other_stream_and_graph():
    # On a stream of its own, and captured: every replay follows the input's present contents.
    torch = _torch()
    mx4 = _mx4()
    w, wv = _weights(500, 256, 21)
    side = torch.cuda.Stream()
    x, exact = _values(6, 256, "f32", 22)
    torch.cuda.synchronize()
    y = mx4.matmul(x, w, stream=side)
    side.synchronize()
    want = M.rounded(exact) @ wv.T
    limit = _bound(M.rounded(exact), wv, want, 256, "f32")
    assert (np.abs(y.double().cpu().numpy() - want) <= limit).all()
    held = x.clone()
    out = torch.empty((6, 500), device="cuda")
    graph = torch.cuda.CUDAGraph()
    mx4.matmul(held, w, out=out)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        mx4.matmul(held, w, out=out)
    for seed in range(4):
        x, _ = _values(6, 256, "f32", 100 + seed)
        held.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mx4.matmul(x, w))
        torch.cuda.synchronize()


def test_refusals():
    torch = _torch()
    mx4 = _mx4()
    w, _ = _weights(40, 64, 1)
    x = torch.zeros(3, 64, device="cuda")
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        mx4.Mx4Matrix.quantize(x.double())
    with pytest.raises(ValueError, match="must not be empty"):
        mx4.Mx4Matrix.quantize(x[:0])
    with pytest.raises(ValueError, match="adjacent"):
        mx4.Mx4Matrix.quantize(x.t())
    with pytest.raises(ValueError, match="device"):
        mx4.Mx4Matrix.quantize(torch.zeros(3, 64))
    with pytest.raises(ValueError, match="64"):
        mx4.matmul(x[:, :63], w)
    with pytest.raises(ValueError, match="bias"):
        mx4.matmul(x, w, bias=torch.zeros(41, device="cuda"))
    with pytest.raises(ValueError, match="shape"):
        mx4.matmul(x, w, out=torch.zeros(3, 41, device="cuda"))
    with pytest.raises(ValueError, match="out is"):
        mx4.Mx4Matrix.quantize(x, out=w)
    with pytest.raises(ValueError, match="codes must have shape"):
        mx4.Mx4Matrix.from_rowmajor(torch.zeros(4, 8, dtype=torch.uint8, device="cuda"),
                                    torch.zeros(4, 1, dtype=torch.uint8, device="cuda"), 32)


@pytest.mark.parametrize("k", [96, 256, 300, 520, 1100])
@pytest.mark.parametrize("rows,n,out", [(300, 6001, "bf16"), (1000, 12500, "f32"), (1000, 12501, "f16")])
def test_product_in_tiles(rows, n, k, out):
    # More tiles of 128 x 128 than half the units: the staged kernels, small tiles and large ones, over one to
    # nine panels of k.
    _check_product(rows, n, k, TYPES[k % 3], out, k == 300)


@pytest.mark.parametrize("rows,n", [(300, 6001), (1000, 12501)])
def test_exact_sums_in_tiles(rows, n):
    # As test_exact_sums: multiples of 1/4 far below 2^24 leave nothing to round.
    torch = _torch()
    k = 1000
    rng = np.random.default_rng(rows)
    codes = rng.integers(0, 16, (rows, 32 * 32), dtype=np.uint8)
    ones = np.full((rows, 32), 127, dtype=np.uint8)
    x = _mx4().Mx4Matrix.from_rowmajor(torch.from_numpy(M.packed(codes)).cuda(), torch.from_numpy(ones).cuda(), k)
    w, wv = _weights(n, k, 3, 127, 128)
    got = _mx4().matmul(x, w).cpu().numpy().astype(np.float64)
    assert np.array_equal(got, M.values(codes, ones, k) @ wv.T)


@pytest.mark.parametrize("rows,n,k", [(1, 333, 7680), (2, 70, 8200), (3, 5000, 7000), (16, 200, 1536), (17, 90, 1400), (32, 150, 700),
                                      (40, 400, 500), (48, 77, 512), (64, 130, 384), (64, 130, 385)])
def test_quantised_in_the_product(rows, n, k):
    # The most rows and columns that the product's own launch quantises, and the next ones.
    for dtype in TYPES:
        _check_product(rows, n, k, dtype, "f32", False)


def test_infinities_and_zeros_quantised_in_the_product():
    torch = _torch()
    x = torch.zeros(20, 300, device="cuda")
    x[3] = torch.linspace(-4, 4, 300, device="cuda")
    x[17, 299] = float("-inf")
    w, wv = _weights(90, 300, 2)
    got = _mx4().matmul(x, w).cpu().numpy()
    assert np.isnan(got[17]).all()
    rest = np.delete(np.arange(20), [3, 17])
    assert (got[rest] == 0).all()
    want = M.rounded(x[3:4].double().cpu().numpy()) @ wv.T
    assert (np.abs(got[3] - want[0]) <= _bound(M.rounded(x[3:4].double().cpu().numpy()), wv, want, 300, "f32")).all()


@pytest.mark.parametrize("rows,cols", [(1, 8200), (63, 129), (200, 70), (64, 128), (129, 1025)])
@pytest.mark.parametrize("dtype", TYPES)
def test_conversion_leaves_the_surroundings(rows, cols, dtype):
    # Buffers with a margin on either side, at addresses that are aligned to an element only.
    torch = _torch()
    x, exact = _values(rows, cols, dtype, cols, spread=0.5)
    m = _mx4().Mx4Matrix.quantize(x)
    flat = torch.full((rows * (cols + 3) + 9,), 3.0, device="cuda", dtype=_dtype(dtype))
    view = torch.as_strided(flat, (rows, cols), (cols + 3, 1), 5)
    m.dequantize(out=view)
    want = torch.from_numpy(M.rounded(exact)).to(_dtype(dtype))
    assert torch.equal(view.cpu(), want)
    view.fill_(3.0)
    assert (flat == 3.0).all()


def test_weights_past_32_bits():
    # 4.6 GB of codes: the last rows' panels lie past 2^32 bytes.
    torch = _torch()
    mx4 = _mx4()
    n, k = 280_001, 32768
    x = torch.zeros((n, k), dtype=torch.bfloat16, device="cuda")
    x[-1] = 1.0
    x[-130, 5] = -3.0
    w = mx4.Mx4Matrix.quantize(x)
    assert w.codes.numel() > 2 ** 32
    for rows in (1, 70, 300):
        got = mx4.matmul(torch.full((rows, k), 0.5, dtype=torch.bfloat16, device="cuda"), w)
        assert (got[:, -1] == k / 2).all() and (got[:, -130] == -1.5).all()
        assert int((got != 0).sum()) == 2 * rows
        del got
    x.zero_()
    w.dequantize(out=x)
    assert (x[-1] == 1.0).all() and float(x[-130, 5]) == -3.0 and int((x[-200:] != 0).sum()) == k + 1


@pytest.mark.parametrize("rows,n,k", [(64, 1000, 256), (64, 1000, 384), (50, 517, 300), (48, 800, 512), (33, 1300, 640), (32, 900, 768),
                                      (17, 51000, 1000), (24, 49999, 900), (9, 50000, 1500), (3, 52000, 7000)])
def test_sums_of_every_panel_of_a_workgroup(rows, n, k):
    # Slices of k are added up in LDS: each of a workgroup's panels of W, its last one too, has its place there.
    _check_product(rows, n, k, TYPES[(rows + k) % 3], "f32", False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,n,at", [(1, 896, 896, 0), (8, 1024, 1024, 0), (24, 800, 800, 0), (64, 384, 384, 0), (16, 512, 700, 40),
                                         (3, 700, 512, -90), (40, 2000, 2000, 0), (200, 300, 300, 0), (300, 6001, 6001, 0)])
def test_result_on_its_own_input(rows, k, n, at, dtype):
    # The product into the buffer that holds x: the same rows, or columns that lie across them. Whatever a row's
    # workgroups write, all of them have read x before.
    torch = _torch()
    w, _ = _weights(n, k, n + at)
    x, _ = _values(rows, k, dtype, rows + k)
    want = _mx4().matmul(x, w, dtype=_dtype(dtype))
    wide = torch.full((rows, max(k, n) + 2 * abs(at)), 3.0, device="cuda", dtype=_dtype(dtype))
    for _ in range(3):
        first = abs(at)
        held = wide[:, first:first + k]
        held.copy_(x)
        got = _mx4().matmul(held, w, out=wide[:, first + at:first + at + n])
        assert torch.equal(got, want)


def test_result_beside_its_input_and_bias():
    # Views of one buffer that share none of its elements.
    torch = _torch()
    w, _ = _weights(96, 160, 3)
    x, _ = _values(9, 160, "f32", 4)
    bias = torch.randn(96, device="cuda")
    want = _mx4().matmul(x, w, bias=bias)
    wide = torch.zeros((9, 160 + 96 + 96), device="cuda")
    wide[:, :160] = x
    wide[4, 256:] = bias
    got = _mx4().matmul(wide[:, :160], w, bias=wide[4, 256:], out=wide[:, 160:256])
    assert torch.equal(got, want) and torch.equal(wide[:, :160], x)
    held = _mx4().Mx4Matrix.quantize(x)
    assert torch.equal(_mx4().matmul(held, w, bias=wide[4, 256:], out=wide[:, 160:256]), want)


def test_tensors_past_32_bits_are_refused():
    # More rows or columns than the C entries' 32-bit sizes hold, which would be taken modulo 2^32.
    torch = _torch()
    from tabby_amd import beam
    mx4 = _mx4()
    flat = torch.empty(2 ** 32 + 3, dtype=torch.float16, device="cuda")
    for x in (flat.view(-1, 1), flat):
        with pytest.raises(ValueError, match="32 bits"):
            mx4.Mx4Matrix.quantize(x)
    w, _ = _weights(4, 3, 1)
    with pytest.raises(ValueError, match="32 bits"):
        mx4.matmul(flat.view(1, -1), w)
    scores = torch.zeros((1, 1), device="cuda")
    with pytest.raises(ValueError, match="32 bits"):
        beam.BeamSelect(vocab_max=3)(flat.view(1, -1), scores, 1)
    with pytest.raises(ValueError, match="32 bits"):
        beam.BeamSelect(vocab_max=3)(flat[:3].view(1, -1), scores, 1, pad_id=2 ** 32)
    parents = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="32 bits"):
        beam.reorder_states([flat.view(1, -1, 1, 1)], parents)
