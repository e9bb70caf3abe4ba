"""The FP8 operators against their definition in 64 bits (fp8_oracle): conversion and the way back
bit for bit, the product within its accumulation's bound, at odd sizes, strides and types, and with
blocks that hold zeros, subnormals, infinities and NaN."""
import numpy as np
import pytest

import fp8_oracle as F
from tabby_amd import sampler as S

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16"]


def _torch():
    import torch
    assert torch.cuda.is_available(), "needs an MI355X"
    return torch


def _fp8():
    from tabby_amd import fp8
    return fp8


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


def _same(got, want):
    return np.array_equal(got, want, equal_nan=True)


def _to(values, dtype):
    """float64 values that f32 holds, rounded to a type, as float64."""
    return _torch().from_numpy(values).to(_dtype(dtype)).double().numpy()


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (1, 128), (2, 129), (15, 127), (63, 256), (64, 96), (65, 1000),
                                       (127, 140), (128, 128), (129, 300), (192, 100), (260, 385)])
def test_round_trip(rows, cols, dtype, block_rows):
    x, exact = _values(rows, cols, dtype, rows * 10007 + cols)
    print(f"round trip {rows} x {cols} {dtype} blocks of {block_rows}", flush=True)
    m = _fp8().Fp8Matrix.quantize(x, block_rows=block_rows)
    want = F.rounded(exact, block_rows)
    for back in TYPES:
        got = m.dequantize(_dtype(back)).double().cpu().numpy()
        assert got.shape == (rows, cols)
        held = _to(want, back)
        assert _same(got, held), (back, np.argwhere(got != held)[:4])
        if back != "f16":
            assert _same(got, want)  # four bits of a significand always fit


def test_every_code_and_every_tie():
    # Blocks led by 448 * 2^E have the scale 2^E: every code, every midpoint of both signs, and the midpoints'
    # neighbours in f32, over many powers.
    torch = _torch()
    near = [v for m in F.MIDDLES.astype(np.float32) for v in (np.nextafter(m, np.float32(0)), m, np.nextafter(m, np.float32(999)))]
    pool = np.array(list(F.LEVELS) + near + [2.0 ** -10, 2.0 ** -11, 2.0 ** -30], dtype=np.float32)
    pool = np.concatenate([pool, -pool])
    rows = []
    for e in (-126, -110, -24, -3, 0, 1, 17, 80, 119):
        for i in range(0, len(pool), 127):
            part = np.zeros(128, dtype=np.float32)
            part[0] = 448.0
            part[1:1 + len(pool[i:i + 127])] = pool[i:i + 127]
            rows.append(np.ldexp(part.astype(np.float64), e).astype(np.float32))
    x = np.stack(rows)
    for block_rows in (1, 128):
        got = _fp8().Fp8Matrix.quantize(torch.from_numpy(x).cuda(), block_rows=block_rows).dequantize().double().cpu().numpy()
        want = _to(F.rounded(x, block_rows), "f32")
        assert _same(got, want), [(x[i, j], got[i, j], want[i, j]) for i, j in np.argwhere(got != want)[:6]]


def test_scales_at_both_ends():
    # The scale is held to 2^-126 and above: subnormals below 448 * 2^-126, f32's largest values; and either side of
    # a change of the power, at 448 * 2^E.
    torch = _torch()
    x = np.zeros((12, 256), dtype=np.float32)
    x[0, :4] = [1e-45, -1e-45, 0, 0]
    x[1, :4] = [2.0 ** -126, 2.0 ** -127, 2.0 ** -135, 2.0 ** -136]
    x[2, :4] = [448 * 2.0 ** -126, 2.0 ** -126, -(2.0 ** -127), 2.0 ** -149]
    x[3, :4] = [np.finfo(np.float32).max, 2.0 ** 127, -(2.0 ** 110), 1.0]
    x[4, 128:132] = [449 * 2.0 ** -126, 2.0 ** -125, 1.5 * 2.0 ** -126, 2.0 ** -127]
    x[5, 0], x[5, 140] = np.inf, 3.0
    x[6, 127], x[6, 1] = np.nan, 5.0
    x[7, 2], x[7, 3] = -np.inf, np.nan
    x[8, :3] = [448.0, 1.0, -0.3]
    x[9, :3] = [np.nextafter(np.float32(448), np.float32(999)), 1.0, -0.3]
    x[10, :3] = [256.0, 1.0, -0.3]
    x[11, :3] = [-0.0, 0.0, -0.0]
    got = _fp8().Fp8Matrix.quantize(torch.from_numpy(x).cuda()).dequantize().double().cpu().numpy()
    want = _to(F.rounded(x), "f32")  # the largest f32 rounds to 256 * 2^120 = 2^128: infinity in f32
    assert np.isinf(want[3, 0])
    assert _same(got, want), [(i, j, x[i, j], got[i, j], want[i, j]) for i, j in np.argwhere((got != want) & ~np.isnan(want))[:8]]
    assert np.isnan(got[5, :128]).all() and not np.isnan(got[5, 128:]).any()
    assert _same(np.signbit(got[11, :3]), np.signbit(x[11, :3]))


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_unaligned_rows(dtype, block_rows):
    torch = _torch()
    base, exact = _values(140, 700, dtype, 5)
    for lo, cols in ((0, 640), (1, 333), (3, 64), (8, 257)):
        x = base[:, lo:lo + cols]
        held = torch.full((140, 800), 7.0, device="cuda")
        got = _fp8().Fp8Matrix.quantize(x, block_rows=block_rows).dequantize(out=held[:, 5:5 + cols])
        assert _same(got.double().cpu().numpy(), F.rounded(exact[:, lo:lo + cols], block_rows)), (lo, cols)
        assert (held[:, :5] == 7.0).all() and (held[:, 5 + cols:] == 7.0).all()
    odd = torch.full((140, 801), 7.0, device="cuda", dtype=_dtype(dtype))
    _fp8().Fp8Matrix.quantize(base[:, :640], block_rows=block_rows).dequantize(out=odd[:, 80:720])
    assert _same(odd[:, 80:720].double().cpu().numpy(), _to(F.rounded(exact[:, :640], block_rows), dtype))
    assert (odd[:, :80] == 7.0).all() and (odd[:, 720:] == 7.0).all()  # nothing beside the rows is written


@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 31), (64, 128), (65, 100), (128, 256), (300, 896), (7, 1027), (129, 144)])
def test_checkpoint_layout(rows, cols):
    # Every code, those of NaN too, and scales of any value.
    torch = _torch()
    rng = np.random.default_rng(rows + cols)
    codes = rng.integers(0, 256, (rows, cols), dtype=np.uint8)
    scales = np.exp(3 * rng.normal(size=(-(-rows // 128), -(-cols // 128)))).astype(np.float32)
    scales[0, 0] = 0.1
    dev = torch.from_numpy(codes).cuda()
    m = _fp8().Fp8Matrix.from_rowmajor(dev, torch.from_numpy(scales).cuda())
    each = scales.repeat(128, 0)[:rows].repeat(128, 1)[:, :cols]
    want = (F.decoded(codes) * each).astype(np.float32)  # one rounding: the product is exact in 64 bits
    assert _same(m.dequantize().cpu().numpy(), want)
    typed = _fp8().Fp8Matrix.from_rowmajor(dev.view(torch.float8_e4m3fn), torch.from_numpy(scales).cuda())
    assert torch.equal(typed.codes, m.codes)


def test_codes_at_an_odd_address():
    torch = _torch()
    rng = np.random.default_rng(3)
    flat = torch.from_numpy(rng.integers(0, 120, 5 + 70 * 300, dtype=np.uint8)).cuda()
    scales = torch.ones((1, 3), device="cuda")
    for lo in (1, 2, 5):
        codes = flat[lo:lo + 70 * 300].view(70, 300)
        got = _fp8().Fp8Matrix.from_rowmajor(codes, scales).dequantize().double().cpu().numpy()
        assert _same(got, F.decoded(codes.cpu().numpy()))


def test_buffers_are_written_again():
    a, _ = _values(50, 200, "f32", 1)
    b, exact = _values(50, 200, "bf16", 2)
    for block_rows in (1, 128):
        m = _fp8().Fp8Matrix.quantize(a, block_rows=block_rows)
        assert _fp8().Fp8Matrix.quantize(b, block_rows=block_rows, out=m) is m
        assert _same(m.dequantize().double().cpu().numpy(), F.rounded(exact, block_rows))


def _weights(n, k, seed, powers=False):
    """(Fp8Matrix, float64 values) of random codes; scales of any value, or powers of two."""
    torch = _torch()
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 127, (n, k), dtype=np.uint8) | (rng.integers(0, 2, (n, k), dtype=np.uint8) << 7)
    shape = (-(-n // 128), -(-k // 128))
    scales = np.exp2(rng.integers(-9, -5, shape)) if powers else np.exp(rng.normal(size=shape)) * 0.01
    scales = scales.astype(np.float32)
    m = _fp8().Fp8Matrix.from_rowmajor(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda())
    return m, F.decoded(codes) * scales.astype(np.float64).repeat(128, 0)[:n].repeat(128, 1)[:, :k]


def _in_tiles(rows, n, out):
    """Whether the product adds codes eight at a time: more than 64 rows, f16 or bf16."""
    return out != "f32" and rows > 64


def _bound(x, w, y, k, out, bias=None):
    """Accumulation in f32, at most one step of 2^-23 relative to an add: k of a block's products, and to each block
    the product of its scales and its addition, and the bias's; then one rounding to the output's type. Where codes are
    added eight at a time, each but the largest loses less than 2^-13 of that one: seven times that of the sum of the magnitudes."""
    torch = _torch()
    grown = np.abs(x) @ np.abs(w).T + (0 if bias is None else np.abs(bias))
    sums = (k + 2 * -(-k // 128) + 1) * 2.0 ** -23 * grown
    if _in_tiles(x.shape[0], w.shape[0], out):
        sums = sums + 7 * 2.0 ** -13 * grown
    eps, tiny = torch.finfo(_dtype(out)).eps, torch.finfo(_dtype(out)).smallest_normal
    return sums + eps / 2 * (np.abs(y) + sums) + tiny * eps


def _check_product(rows, n, k, dtype, out, bias, seed=0):
    torch = _torch()
    x, exact = _values(rows, k, dtype, 31 * rows + n + seed, spread=0.3)
    w, wv = _weights(n, k, 7 * n + k + seed)
    b = np.random.default_rng(n).normal(size=n).astype(np.float32) if bias else None
    head = _fp8().LmHeadFp8(w, None if b is None else torch.from_numpy(b).cuda())
    print(f"product {rows} x {n} x {k} {dtype}->{out} bias={bias}", flush=True)
    xv = F.rounded(exact)
    want = xv @ wv.T + (0 if b is None else b.astype(np.float64))
    limit = _bound(xv, wv, want, k, out, b)
    got = head.logits(x, dtype=_dtype(out))
    assert got.shape == (rows, n) and got.dtype == _dtype(out)
    got = got.double().cpu().numpy()
    if out == "f16":
        limit = np.where(np.abs(want) > 65000, np.inf, limit)  # near the end of its range, or past it
        got = np.where(np.isinf(got) & (np.abs(want) > 65000), want, got)
    err = np.abs(got - want)
    assert (err <= limit).all(), (err.max(), np.argwhere(~(err <= limit))[:4])
    first = head.logits(x, dtype=_dtype(out))
    again = _fp8().matmul(_fp8().Fp8Matrix.quantize(x), w, head.bias, dtype=_dtype(out))
    assert torch.equal(first, again)  # quantised in the call or before it


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 64, 128), (1, 1000, 896), (2, 63, 31), (3, 65, 160), (15, 17, 33),
                                      (16, 200, 1024), (17, 129, 257), (31, 96, 64), (33, 300, 800), (48, 77, 500), (64, 64, 4096),
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


@pytest.mark.parametrize("k", [96, 256, 300, 520, 1100])
@pytest.mark.parametrize("rows,n,out", [(300, 6001, "bf16"), (1000, 12500, "f32"), (1000, 12501, "f16")])
def test_product_in_tiles(rows, n, k, out):
    # More tiles of 128 x 128 than half the units: the staged kernels, small tiles and large ones, over one to
    # nine panels of k.
    _check_product(rows, n, k, TYPES[k % 3], out, k == 300)


@pytest.mark.parametrize("rows,n", [(1, 700), (5, 700), (16, 700), (40, 700), (70, 700), (260, 700), (300, 6001), (1000, 12501)])
def test_exact_sums(rows, n):
    # Whole numbers up to 16 and scales of one: every sum is a whole number below 2^24, whatever the order.
    torch = _torch()
    k = 1500
    rng = np.random.default_rng(rows)
    x = rng.integers(-16, 17, (rows, k)).astype(np.float32)
    x[:, ::128] = 448.0  # the scale of every block is 1
    w = rng.integers(-16, 17, (n, k)).astype(np.float64)
    codes = (F.nearest(np.abs(w)) | (np.signbit(w).astype(np.int64) << 7)).astype(np.uint8)
    assert np.array_equal(F.decoded(codes), w)
    m = _fp8().Fp8Matrix.from_rowmajor(torch.from_numpy(codes).cuda(), torch.ones((-(-n // 128), 12), device="cuda"))
    got = _fp8().matmul(torch.from_numpy(x).cuda(), m).double().cpu().numpy()
    assert np.array_equal(got, x.astype(np.float64) @ w.T)


@pytest.mark.parametrize("rows,n", [(70, 330), (300, 6001), (1000, 12501)])
def test_each_block_has_its_own_scale(rows, n):
    # One block of each row of x nonzero, with a power of its own, and a power of its own to every block of the
    # weights: a value or scale taken from another block, row or tile shows.
    torch = _torch()
    k = 1200
    rng = np.random.default_rng(1)
    x = np.zeros((rows, k))
    for r in range(rows):
        b = r % 10
        x[r, 128 * b:128 * b + 12] = rng.choice([-1.0, 1.0, 2.0, 3.0], 12) * 2.0 ** (r % 7)
    codes = (F.nearest(rng.choice([1.0, 0.5, 1.5, 2.0], (n, k)))).astype(np.uint8)
    scales = np.exp2(rng.integers(-8, 9, (-(-n // 128), 10))).astype(np.float32)
    m = _fp8().Fp8Matrix.from_rowmajor(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda())
    wv = F.decoded(codes) * scales.astype(np.float64).repeat(128, 0)[:n].repeat(128, 1)[:, :k]
    got = _fp8().matmul(torch.from_numpy(x).float().cuda(), m).double().cpu().numpy()
    assert np.array_equal(got, x @ wv.T)


@pytest.mark.parametrize("rows", [2, 20, 90, 300])
def test_nan_blocks_reach_their_rows_alone(rows):
    torch = _torch()
    n = 6001 if rows == 300 else 400
    x, exact = _values(rows, 300, "f32", 3)
    x[1, 290] = float("inf")
    w, wv = _weights(n, 300, 4)
    got = _fp8().matmul(x, w).cpu().numpy()
    assert np.isnan(got[1]).all()
    assert np.isfinite(np.delete(got, 1, 0)).all()
    wv[200, 5] = np.nan  # a weight that is none: its block of 128 rows
    wq = _fp8().Fp8Matrix.quantize(torch.from_numpy(wv).float().cuda(), block_rows=128)
    x[1, 290] = 0.0
    got = _fp8().matmul(x, wq).cpu().numpy()
    assert np.isnan(got[:, 128:256]).all() and np.isfinite(np.delete(got, np.arange(128, 256), 1)).all()


@pytest.mark.parametrize("rows", [1, 30, 140])
def test_product_into_strided_output(rows):
    torch = _torch()
    x, exact = _values(rows, 320, "bf16", 9)
    w, wv = _weights(203, 320, 10, powers=True)
    for out in TYPES:
        wide = torch.full((rows, 300), 5.0, device="cuda", dtype=_dtype(out))
        for lo in (0, 1, 4, 7):
            wide.fill_(5.0)
            _fp8().matmul(x, w, out=wide[:, lo:lo + 203])
            want = F.rounded(exact) @ wv.T
            err = np.abs(wide[:, lo:lo + 203].double().cpu().numpy() - want)
            assert (err <= _bound(F.rounded(exact), wv, want, 320, out)).all()
            assert (wide[:, :lo] == 5.0).all() and (wide[:, lo + 203:] == 5.0).all()


def test_other_stream_and_graph():
    # On a stream of its own, and captured: every replay follows the input's present contents.
    torch = _torch()
    fp8 = _fp8()
    w, wv = _weights(500, 256, 21)
    side = torch.cuda.Stream()
    x, exact = _values(6, 256, "f32", 22)
    torch.cuda.synchronize()
    y = fp8.matmul(x, w, stream=side)
    side.synchronize()
    want = F.rounded(exact) @ wv.T
    limit = _bound(F.rounded(exact), wv, want, 256, "f32")
    assert (np.abs(y.double().cpu().numpy() - want) <= limit).all()
    held = x.clone()
    out = torch.empty((6, 500), device="cuda")
    matrix = fp8.Fp8Matrix(6, 256)
    graph = torch.cuda.CUDAGraph()
    fp8.matmul(held, w, out=out)
    fp8.Fp8Matrix.quantize(held, out=matrix)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        fp8.matmul(held, w, out=out)
        fp8.Fp8Matrix.quantize(held, out=matrix)
    for seed in range(4):
        x, exact = _values(6, 256, "f32", 100 + seed)
        held.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fp8.matmul(x, w))
        assert _same(matrix.dequantize().double().cpu().numpy(), F.rounded(exact))
        torch.cuda.synchronize()


def test_refusals():
    torch = _torch()
    fp8 = _fp8()
    w, _ = _weights(40, 64, 1)
    x = torch.zeros(3, 64, device="cuda")
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        fp8.Fp8Matrix.quantize(x.double())
    with pytest.raises(ValueError, match="must not be empty"):
        fp8.Fp8Matrix.quantize(x[:0])
    with pytest.raises(ValueError, match="adjacent"):
        fp8.Fp8Matrix.quantize(x.t())
    with pytest.raises(ValueError, match="device"):
        fp8.Fp8Matrix.quantize(torch.zeros(3, 64))
    with pytest.raises(S.SamplingError, match="block_rows must be 1 or 128, got 64"):
        fp8.Fp8Matrix.quantize(x, block_rows=64)
    with pytest.raises(ValueError, match="64"):
        fp8.matmul(x[:, :63], w)
    with pytest.raises(ValueError, match="bias"):
        fp8.matmul(x, w, bias=torch.zeros(41, device="cuda"))
    with pytest.raises(ValueError, match="shape"):
        fp8.matmul(x, w, out=torch.zeros(3, 41, device="cuda"))
    with pytest.raises(ValueError, match="out is"):
        fp8.Fp8Matrix.quantize(x, out=w)
    rows = fp8.Fp8Matrix.quantize(x)
    with pytest.raises(ValueError, match="weights must have blocks of 128"):
        fp8.matmul(x, rows)
    with pytest.raises(ValueError, match="weights must have blocks of 128"):
        fp8.LmHeadFp8(rows)
    with pytest.raises(ValueError, match="blocks of one row"):
        fp8.matmul(w, w)
    with pytest.raises(ValueError, match="scales must have shape"):
        fp8.Fp8Matrix.from_rowmajor(torch.zeros(4, 8, dtype=torch.uint8, device="cuda"), torch.zeros(4, 1, device="cuda"))
    with pytest.raises(ValueError, match="uint8 or float8_e4m3fn"):
        fp8.Fp8Matrix.from_rowmajor(torch.zeros(4, 8, dtype=torch.int8, device="cuda"), torch.zeros(1, 1, device="cuda"))
    with pytest.raises(S.SamplingError, match="overlap"):
        fp8.matmul(rows, w, out=rows.data[:3 * 40 * 4].view(torch.float32).view(3, 40))


def test_weights_past_32_bits():
    # 4.6 GB of codes: the last rows' panels lie past 2^32 bytes.
    torch = _torch()
    fp8 = _fp8()
    n, k = 140_001, 32768
    x = torch.zeros((n, k), dtype=torch.bfloat16, device="cuda")
    x[-1] = 1.0
    x[-130, 5] = -3.0
    w = fp8.Fp8Matrix.quantize(x, block_rows=128)
    assert w.codes.numel() > 2 ** 32
    for rows in (1, 70, 300):
        got = fp8.matmul(torch.full((rows, k), 0.5, dtype=torch.bfloat16, device="cuda"), w)
        assert (got[:, -1] == k / 2).all() and (got[:, -130] == -1.5).all()
        assert int((got != 0).sum()) == 2 * rows
        del got
    x.zero_()
    w.dequantize(out=x)
    assert (x[-1] == 1.0).all() and float(x[-130, 5]) == -3.0 and int((x[-200:] != 0).sum()) == k + 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,n,at", [(1, 896, 896, 0), (8, 1024, 1024, 0), (24, 800, 800, 0), (64, 384, 384, 0), (16, 512, 700, 40),
                                         (3, 700, 512, -90), (40, 2000, 2000, 0), (200, 300, 300, 0), (300, 6001, 6001, 0)])
def test_result_on_its_own_input(rows, k, n, at, dtype):
    # The product into the buffer that holds x: the same rows, or columns that lie across them.
    torch = _torch()
    w, _ = _weights(n, k, n + at)
    x, _ = _values(rows, k, dtype, rows + k)
    want = _fp8().matmul(x, w, dtype=_dtype(dtype))
    wide = torch.full((rows, max(k, n) + 2 * abs(at)), 3.0, device="cuda", dtype=_dtype(dtype))
    for _ in range(3):
        first = abs(at)
        held = wide[:, first:first + k]
        held.copy_(x)
        got = _fp8().matmul(held, w, out=wide[:, first + at:first + at + n])
        assert torch.equal(got, want)


@pytest.mark.parametrize("rows,n,k", [(64, 1000, 256), (64, 1000, 384), (50, 517, 300), (48, 800, 512), (33, 1300, 640), (32, 900, 768),
                                      (17, 51000, 1000), (24, 49999, 900), (9, 50000, 1500), (3, 52000, 7000)])
def test_sums_of_every_panel_of_a_workgroup(rows, n, k):
    # Slices of k are added up in LDS: each of a workgroup's panels of W, its last one too, has its place there.
    _check_product(rows, n, k, TYPES[(rows + k) % 3], "f32", False)
