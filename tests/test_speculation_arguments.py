"""The C entries of the FP8 operators and of the verification of drafted tokens refuse bad arguments before any GPU
work: no GPU is needed to be refused. The addresses are never read."""
import ctypes

import pytest

from tabby_amd import sampler as S

A = 1 << 30  # aligned addresses that nothing reads, far apart
B, C, D, E = A << 1, A << 2, A << 3, A << 4


@pytest.fixture(scope="module")
def lib():
    return S.load_library()


def _refused(lib, rc, text, status=S.TABBY_EINVAL):
    assert rc == status
    assert text in lib.tabby_last_error().decode(), lib.tabby_last_error().decode()


def test_fp8_sizes(lib):
    code, scale = ctypes.c_int64(), ctypes.c_int64()
    for rows, cols, block, panels, scales in ((1, 1, 1, 1, 256), (64, 128, 1, 1, 256), (65, 128, 1, 2, 512), (64, 129, 1, 2, 512),
                                              (1, 1, 128, 1, 256), (128, 128, 128, 2, 256), (151936, 896, 128, 2374 * 7, 33280)):
        assert lib.tabby_fp8_bytes(rows, cols, block, ctypes.byref(code), ctypes.byref(scale)) == 0
        assert (code.value, scale.value) == (panels * 8192, scales), (rows, cols, block, code.value, scale.value)
    big = 2 ** 31 - 129
    assert lib.tabby_fp8_bytes(big, big, 1, ctypes.byref(code), ctypes.byref(scale)) == 0
    assert code.value == -(-big // 64) * -(-big // 128) * 8192
    _refused(lib, lib.tabby_fp8_bytes(0, 5, 1, ctypes.byref(code), ctypes.byref(scale)), ">= 1")
    _refused(lib, lib.tabby_fp8_bytes(5, -1, 1, ctypes.byref(code), ctypes.byref(scale)), ">= 1")
    _refused(lib, lib.tabby_fp8_bytes(5, 5, 64, ctypes.byref(code), ctypes.byref(scale)), "block_rows")
    _refused(lib, lib.tabby_fp8_bytes(5, 2 ** 31 - 1, 1, ctypes.byref(code), ctypes.byref(scale)), "padding")
    _refused(lib, lib.tabby_fp8_bytes(5, 5, 1, None, ctypes.byref(scale)), "null")


def test_fp8_conversion_arguments(lib):
    q, d, p = lib.tabby_fp8_quantize_device, lib.tabby_fp8_dequantize_device, lib.tabby_fp8_pack_device
    _refused(lib, q(None, 0, 1, 32, 32, 1, B, C, None), "null")
    _refused(lib, q(A, 0, 1, 32, 32, 1, None, C, None), "null")
    _refused(lib, q(A, 0, 1, 32, 32, 1, B + 8, C, None), "aligned")
    _refused(lib, q(A, 0, 1, 32, 32, 1, B, C + 2, None), "aligned")
    _refused(lib, q(A, 3, 1, 32, 32, 1, B, C, None), "dtype")
    _refused(lib, q(A, 0, 2, 32, 31, 1, B, C, None), "row_stride")
    _refused(lib, q(A + 2, 0, 1, 32, 32, 1, B, C, None), "elements")
    _refused(lib, q(A, 0, 0, 32, 32, 1, B, C, None), ">= 1")
    _refused(lib, q(A, 0, 1, 32, 32, 2, B, C, None), "block_rows")
    _refused(lib, q(A, 0, 1, 32, 32, 1, A, C, None), "overlap")
    _refused(lib, q(A, 0, 65, 32, 32, 1, B, A + 8192, None), "overlap")
    _refused(lib, d(A, B, 1, 32, 1, None, 0, 32, None), "null")
    _refused(lib, d(A, B, 1, 32, 1, C, -1, 32, None), "dtype")
    _refused(lib, d(A, B, 2, 32, 1, C, 0, 5, None), "row_stride")
    _refused(lib, d(A, None, 1, 32, 1, C, 0, 32, None), "null")
    _refused(lib, d(A, B, 1, 32, 1, A, 0, 32, None), "overlap")
    _refused(lib, d(A, B, 1, 32, 3, C, 0, 32, None), "block_rows")
    _refused(lib, p(None, A, 1, 32, B, C, None), "null")
    _refused(lib, p(A, D, 1, 0, B, C, None), ">= 1")
    _refused(lib, p(A, D + 1, 1, 32, B, C, None), "aligned")
    _refused(lib, p(A, D, 1, 32, A, C, None), "overlap")
    _refused(lib, p(A, D, 1, 32, B, D, None), "overlap")


def test_fp8_product_arguments(lib):
    m, f = lib.tabby_fp8_matmul_device, lib.tabby_fp8_linear_device
    _refused(lib, m(A, B, 1, None, D, None, 64, 128, E, 0, 64, None), "null")
    _refused(lib, m(A, B, 1, C, D, None, 64, 0, E, 0, 64, None), ">= 1")
    _refused(lib, m(A, B, 2, C, D, None, 64, 128, E, 0, 63, None), "out_stride")
    _refused(lib, m(A, B, 1, C, D, None, 64, 128, E, 5, 64, None), "dtype")
    _refused(lib, m(A, B, 1, C, D, None, 64, 128, E + 1, 1, 64, None), "elements")
    _refused(lib, m(A, B, 1, C, D, A + 2, 64, 128, E, 0, 64, None), "bias")
    _refused(lib, m(A, B, 1, C, D, None, 64, 128, C, 0, 64, None), "overlap")
    _refused(lib, m(A, B, 1, C, D, None, 64, 128, A, 0, 64, None), "overlap")
    _refused(lib, m(A, B, 1, C, D, E, 64, 128, E, 0, 64, None), "bias")
    size = 8192 + 256
    _refused(lib, f(A, 0, 128, 1, C, D, None, 64, 128, E, 0, 64, None, size, None), "null")
    _refused(lib, f(A, 9, 128, 1, C, D, None, 64, 128, E, 0, 64, B, size, None), "dtype")
    _refused(lib, f(A, 0, 100, 2, C, D, None, 64, 128, E, 0, 64, B, size, None), "x_stride")
    _refused(lib, f(A + 1, 1, 128, 1, C, D, None, 64, 128, E, 0, 64, B, size, None), "elements")
    _refused(lib, f(A, 0, 128, 1, C, D, None, 64, 128, E, 0, 64, B, size - 1, None), "workspace")
    _refused(lib, f(A, 0, 128, 1, C, D, None, 64, 128, E, 0, 64, B + 8, size, None), "workspace")
    _refused(lib, f(A, 0, 128, 1, C, D, None, 64, 128, E, 0, 64, A, size, None), "overlap")
    _refused(lib, f(A, 0, 128, 1, C, D, None, 64, 128, E, 0, 64, E, size, None), "overlap")
    _refused(lib, f(A, 0, 128, 1, C, D, None, 64, 128, E, 0, 64, C, size, None), "overlap")


def test_verification_workspace(lib):
    size = ctypes.c_int64()
    w = lib.tabby_draft_workspace
    _refused(lib, w(0, 4, 100, ctypes.byref(size)), ">= 1")
    _refused(lib, w(1, 4, 0, ctypes.byref(size)), ">= 1")
    _refused(lib, w(1, 64, 100, ctypes.byref(size)), "drafts_max must be between 0 and 63, got 64")
    _refused(lib, w(1, -1, 100, ctypes.byref(size)), "drafts_max")
    _refused(lib, w(1, 4, 2 ** 24 + 1, ctypes.byref(size)), "vocab")
    _refused(lib, w(65536, 0, 100, ctypes.byref(size)), "65535")
    _refused(lib, w(65535, 63, 100, ctypes.byref(size)), "rows")
    _refused(lib, w(1, 4, 100, None), "null")
    # A workspace serves every smaller call.
    def bytes_of(*sizes):
        assert w(*sizes, ctypes.byref(size)) == 0
        return size.value
    shapes = [(1, 0, 1), (1, 4, 151936), (7, 3, 5000), (64, 4, 151936), (100, 63, 2 ** 24), (500, 4, 300), (5000, 0, 1000), (65535, 0, 10)]
    for a in shapes:
        for b in shapes:
            if all(x <= y for x, y in zip(a, b)):
                assert bytes_of(*a) <= bytes_of(*b), (a, b)


def test_verification_arguments(lib):
    size = ctypes.c_int64()
    assert lib.tabby_draft_workspace(3, 2, 1000, ctypes.byref(size)) == 0
    need = size.value
    step = 1 << 30

    def call(logits=step, dtype=0, stride=1000, rows=9, draft=2 * step, draft_stride=1000, drafts=3 * step, uniforms=4 * step, offsets=None,
             requests=3, most=2, vocab=1000, params=5 * step, tokens=6 * step, accepted=7 * step, status=8 * step, space=9 * step,
             bytes_=need, flags=0):
        return lib.tabby_draft_verify_device(logits, dtype, stride, rows, draft, draft_stride, drafts, uniforms, offsets, requests, most,
                                             vocab, params, tokens, accepted, status, space, bytes_, flags, None)
    for name in ("logits", "drafts", "uniforms", "params", "tokens", "accepted", "space"):
        _refused(lib, call(**{name: None}), "null")
    _refused(lib, call(dtype=3), "dtype")
    _refused(lib, call(rows=2), "rows must be between")
    _refused(lib, call(rows=10), "rows must be between")
    _refused(lib, call(rows=8), "without offsets")
    _refused(lib, call(stride=999), "strides")
    _refused(lib, call(draft_stride=999), "strides")
    _refused(lib, call(logits=step + 2), "elements")
    _refused(lib, call(draft=2 * step + 1, dtype=1), "elements")
    for name in ("drafts", "tokens", "accepted", "status"):
        _refused(lib, call(**{name: 10 * step + 2}), "4-byte")
    _refused(lib, call(offsets=10 * step + 1), "4-byte")
    _refused(lib, call(uniforms=4 * step + 4), "8-byte")
    _refused(lib, call(params=5 * step + 4), "8-byte")
    _refused(lib, call(flags=64), "flags")
    _refused(lib, call(bytes_=need - 1), "workspace")
    _refused(lib, call(space=9 * step + 8), "workspace")
    _refused(lib, call(requests=0), ">= 1")
    _refused(lib, call(most=64, rows=3), "drafts_max")
    _refused(lib, call(vocab=2 ** 24 + 1, stride=2 ** 25, draft_stride=2 ** 25), "vocab")
    # What is written lies apart from what is read.
    for name in ("tokens", "accepted", "status", "space"):
        for other in (step, 2 * step, 3 * step, 4 * step, 5 * step):
            _refused(lib, call(**{name: other}), "overlap")
    _refused(lib, call(tokens=7 * step), "overlap")
    _refused(lib, call(status=9 * step + 64), "overlap")
    _refused(lib, call(offsets=6 * step), "overlap")


def test_fast_sums_arguments(lib):
    m, f = lib.tabby_fp8_matmul_device, lib.tabby_fp8_linear_device
    fast = 0x100
    _refused(lib, m(A, B, 1, C, D, None, 64, 128, E, fast | S.TABBY_F32, 64, None), "f16 and bf16 results")
    _refused(lib, f(A, 0, 128, 1, C, D, None, 64, 128, E, fast | S.TABBY_F32, 64, B, 8192 + 256, None), "f16 and bf16 results")
    _refused(lib, m(A, B, 1, C, D, None, 64, 128, E, fast | 3, 64, None), "dtype")
    _refused(lib, m(A, B, 1, C, D, None, 64, 128, E, -1, 64, None), "dtype")
    _refused(lib, m(A, B, 1, C, D, None, 64, 128, E + 1, fast | S.TABBY_BF16, 64, None), "elements")
    _refused(lib, m(A, B, 2, C, D, None, 64, 128, E, fast | S.TABBY_F16, 63, None), "out_stride")
    _refused(lib, f(A, fast, 128, 1, C, D, None, 64, 128, E, 1, 64, B, 8192 + 256, None), "dtype")
