"""The C entries of the MXFP4 and beam operators refuse bad arguments before any GPU work: no
GPU is needed to be refused. The addresses are never read."""
import ctypes

import pytest

from tabby_amd import sampler as S

A = 1 << 20  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    return S.load_library()


def _refused(lib, rc, text, status=S.TABBY_EINVAL):
    assert rc == status
    assert text in lib.tabby_last_error().decode()


def test_mx4_sizes(lib):
    code, scale = ctypes.c_int64(), ctypes.c_int64()
    for rows, cols, panels in ((1, 1, 1), (64, 128, 1), (65, 128, 2), (64, 129, 2), (151936, 896, 2374 * 7)):
        assert lib.tabby_mx4_bytes(rows, cols, ctypes.byref(code), ctypes.byref(scale)) == 0
        assert (code.value, scale.value) == (panels * 4096, panels * 256)
    big = 2 ** 31 - 129
    assert lib.tabby_mx4_bytes(big, big, ctypes.byref(code), ctypes.byref(scale)) == 0
    assert code.value == -(-big // 64) * -(-big // 128) * 4096
    _refused(lib, lib.tabby_mx4_bytes(0, 5, ctypes.byref(code), ctypes.byref(scale)), ">= 1")
    _refused(lib, lib.tabby_mx4_bytes(5, 2 ** 31 - 1, ctypes.byref(code), ctypes.byref(scale)), "padding")
    _refused(lib, lib.tabby_mx4_bytes(5, 5, None, ctypes.byref(scale)), "null")


def test_mx4_conversion_arguments(lib):
    q, d, p = lib.tabby_mx4_quantize_device, lib.tabby_mx4_dequantize_device, lib.tabby_mx4_pack_device
    _refused(lib, q(None, 0, 1, 32, 32, A, A, None), "null")
    _refused(lib, q(A, 0, 1, 32, 32, A + 8, A, None), "aligned")
    _refused(lib, q(A, 0, 1, 32, 32, A, A + 2, None), "aligned")
    _refused(lib, q(A, 3, 1, 32, 32, A, A, None), "dtype")
    _refused(lib, q(A, 0, 2, 32, 31, A, A, None), "row_stride")
    _refused(lib, q(A + 2, 0, 1, 32, 32, A, A, None), "elements")
    _refused(lib, q(A, 0, 0, 32, 32, A, A, None), ">= 1")
    _refused(lib, d(A, A, 1, 32, None, 0, 32, None), "null")
    _refused(lib, d(A, A, 1, 32, A, -1, 32, None), "dtype")
    _refused(lib, d(A, A, 2, 32, A, 0, 5, None), "row_stride")
    _refused(lib, d(A, None, 1, 32, A, 0, 32, None), "null")
    _refused(lib, p(None, A, 1, 32, A, A, None), "null")
    _refused(lib, p(A, A, 1, 0, A, A, None), ">= 1")


def test_mx4_product_arguments(lib):
    m, f = lib.tabby_mx4_matmul_device, lib.tabby_mx4_linear_device
    _refused(lib, m(A, A, 1, None, A, None, 64, 128, A, 0, 64, None), "null")
    _refused(lib, m(A, A, 1, A, A, None, 64, 0, A, 0, 64, None), ">= 1")
    _refused(lib, m(A, A, 2, A, A, None, 64, 128, A, 0, 63, None), "out_stride")
    _refused(lib, m(A, A, 1, A, A, None, 64, 128, A, 5, 64, None), "dtype")
    _refused(lib, m(A, A, 1, A, A, None, 64, 128, A + 1, 1, 64, None), "elements")
    _refused(lib, f(A, 0, 128, 1, A, A, None, 64, 128, A, 0, 64, None, 1 << 20, None), "null")
    _refused(lib, f(A, 9, 128, 1, A, A, None, 64, 128, A, 0, 64, A, 1 << 20, None), "dtype")
    _refused(lib, f(A, 0, 100, 2, A, A, None, 64, 128, A, 0, 64, A, 1 << 20, None), "x_stride")
    _refused(lib, f(A, 0, 128, 1, A, A, None, 64, 128, A, 0, 64, A, 4351, None), "workspace")
    _refused(lib, f(A, 0, 128, 1, A, A, None, 64, 128, A, 0, 64, A + 8, 1 << 20, None), "workspace")


def test_beam_selection_arguments(lib):
    size = ctypes.c_int64()
    _refused(lib, lib.tabby_beam_workspace(1, 65, 10, 4, ctypes.byref(size)), "beams must be between 1 and 64, got 65")
    _refused(lib, lib.tabby_beam_workspace(1, 4, 10, 129, ctypes.byref(size)), "count must be between 1 and 128, got 129")
    _refused(lib, lib.tabby_beam_workspace(0, 4, 10, 4, ctypes.byref(size)), ">= 1")
    assert lib.tabby_beam_workspace(3, 4, 1000, 8, ctypes.byref(size)) == 0
    need = size.value

    def call(logits=A, dtype=0, stride=1000, groups=3, beams=4, vocab=1000, scores=A, pad=0, count=8, tokens=A, space=A,
             bytes_=need):
        return lib.tabby_beam_select_device(logits, dtype, stride, groups, beams, vocab, scores, None, None, pad, count,
                                            tokens, A, A, None, space, bytes_, None)
    _refused(lib, call(logits=None), "null")
    _refused(lib, call(scores=None), "null")
    _refused(lib, call(space=None), "null")
    _refused(lib, call(dtype=7), "dtype")
    _refused(lib, call(stride=999), "row_stride")
    _refused(lib, call(logits=A + 2), "elements")
    _refused(lib, call(pad=-1), "pad_id")
    _refused(lib, call(count=0), "count")
    _refused(lib, call(vocab=0), ">= 1")
    _refused(lib, call(groups=2 ** 26, beams=64), "32 bits")
    _refused(lib, call(bytes_=need - 1), "workspace")
    _refused(lib, call(space=A + 8), "workspace")


def test_beam_reorder_arguments(lib):
    def call(src=(A, 2 * A), dst=(3 * A, 4 * A), groups=2, beams=4, segments=2, capacity=16, unit=128, row=4096, segment=2048,
             parents=A):
        n = len(src)
        arr = ctypes.c_void_p * n
        return lib.tabby_beam_reorder_device(arr(*src), arr(*dst), n, groups, beams, segments, capacity, unit, row, segment,
                                             parents, None, None)
    _refused(lib, call(parents=None), "null")
    _refused(lib, call(src=(A, None)), "null")
    _refused(lib, call(beams=65), "beams must be between 1 and 64, got 65")
    _refused(lib, call(capacity=0), ">= 1")
    _refused(lib, call(unit=0), ">= 1")
    _refused(lib, call(segment=2047), "segment_stride")
    _refused(lib, call(row=4095), "row_stride")
    _refused(lib, call(capacity=2 ** 62, unit=8), "63 bits")
    _refused(lib, call(dst=(A, 4 * A)), "in place")
    _refused(lib, call(dst=(A + 4096, 4 * A)), "overlap")
    _refused(lib, call(groups=2 ** 20, segments=2 ** 20), "32 bits")


def test_mx4_results_apart_from_operands(lib):
    # 1 x 32 and 64 x 128: one panel, 4,096 bytes of codes and 256 of scales. B, C, ... lie 1 MiB apart.
    B, C, D, E = (A * i for i in (2, 3, 4, 5))
    q, d, p = lib.tabby_mx4_quantize_device, lib.tabby_mx4_dequantize_device, lib.tabby_mx4_pack_device
    m, f = lib.tabby_mx4_matmul_device, lib.tabby_mx4_linear_device
    _refused(lib, q(A, 0, 1, 32, 32, A, B, None), "overlap")
    _refused(lib, q(A, 0, 1, 32, 32, A - 4080, B, None), "overlap")
    _refused(lib, q(A, 0, 1, 32, 32, B, A + 124, None), "overlap")
    _refused(lib, q(A, 0, 3, 32, 2 ** 20, A + 8 * 2 ** 20 + 112, 64 * A, None), "overlap")  # the last row
    _refused(lib, d(A, B, 1, 32, A + 4092, 0, 32, None), "overlap")
    _refused(lib, d(A, B, 1, 32, B, 0, 32, None), "overlap")
    _refused(lib, p(A, B, 1, 32, A, C, None), "overlap")
    _refused(lib, p(A, B, 1, 32, C, B, None), "overlap")
    _refused(lib, m(A, B, 1, C, D, None, 64, 128, A, 0, 64, None), "overlap")
    _refused(lib, m(A, B, 1, C, D, None, 64, 128, D + 252, 0, 64, None), "overlap")
    _refused(lib, m(A, B, 1, C, D, E, 64, 128, E + 252, 0, 64, None), "overlap")
    _refused(lib, f(A, 0, 128, 1, C, D, None, 64, 128, C, 0, 64, E, 4352, None), "overlap")
    _refused(lib, f(A, 0, 128, 1, C, D, B, 64, 128, B, 0, 64, E, 4352, None), "overlap")
    _refused(lib, f(A, 0, 128, 1, C, D, None, 64, 128, E + 4348, 0, 64, E, 4352, None), "workspace")
    _refused(lib, f(A, 0, 128, 1, C, D, None, 64, 128, B, 0, 64, A, 4352, None), "workspace")
    _refused(lib, f(A, 0, 128, 1, C, D, None, 64, 128, B, 0, 64, C, 4352, None), "overlap")


def test_beam_reorder_states_apart(lib):
    def call(src, dst=None, groups=2, beams=4, segments=2, capacity=16, unit=128, row=4096, segment=2048):
        dst = src if dst is None else dst
        n = len(src)
        arr = ctypes.c_void_p * n
        return lib.tabby_beam_reorder_device(arr(*src), arr(*dst), n, groups, beams, segments, capacity, unit, row, segment, A,
                                             None, None)
    span = 8 * 4096
    far = [A * (i + 2) for i in range(200)]
    for src, dst in (((A, A), None),                                      # a cache listed twice
                     ((A, 2 * A, 3 * A, 2 * A), None),
                     ((A, A + span - 16), None),
                     ((2 * A + 4096, 2 * A), None),
                     ((A, 2 * A), (3 * A, A)),                            # one's destination is another's source
                     ((A, 2 * A), (3 * A, 2 * A + 2048)),
                     ((A, 2 * A), (3 * A, 3 * A)),                        # two destinations
                     (tuple(far) + (far[77],), None),
                     (tuple(far), tuple(a + 200 * A for a in far[:-1]) + (far[3],))):
        _refused(lib, call(src, dst), "overlap")
    # Between the segments and rows of one another, but for one byte.
    _refused(lib, call((A, A + 1023), segments=3, capacity=1024, unit=1, row=16384, segment=2048), "overlap")
    _refused(lib, call((A, A + 16384 * 2 + 3 * 2048 - 1), segments=4, capacity=2048, unit=1, row=16384, segment=4096), "overlap")
    _refused(lib, call((A, A + 63), beams=1, groups=1, segments=9, capacity=64, unit=1, segment=128, row=0), "overlap")
