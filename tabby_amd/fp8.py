"""8-bit floating point (e4m3) with a scale for each block of 128 on the GPU: conversion, the way
back, and the product of activations with such weights, over the C ABI's ``tabby_fp8_*`` entries.

It stands beside ``mx4`` and ``sampler.LmHeadQ4`` (the reference's int4 lm_head, src/engine/
forward.ts:408-428, 732-770) for checkpoints whose weights are FP8: e4m3 codes, and a float32 scale
to each square block of 128 x 128. Activations have a scale to each 128 values of a row;
``LmHeadFp8.logits`` quantises the hidden states in the call.

Every call is asynchronous on the given stream (default: torch's current one) and checks its
arguments before any GPU work.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from .mx4 import INT32_MAX, _result_code, call_on, dtype_code, on_device, rows_of
from .sampler import _check, load_library

FAST_SUMS = 0x100  # TABBY_FP8_FAST_SUMS
BLOCK = 128  # columns to a scale, and rows of a weight's block
PANEL_ROWS, PANEL_COLS = 64, 128  # a panel's codes take 8,192 bytes, the scales of its rows 256


def sizes(rows: int, cols: int, block_rows: int):
    """Bytes of a matrix's codes and scales."""
    if rows > INT32_MAX or cols > INT32_MAX:
        raise ValueError(f"rows and columns must fit 32 bits, got {rows} x {cols}")
    if 0 < rows < 2 ** 20 and 0 < cols < 2 ** 20 and block_rows == 1:
        panels = -(-rows // PANEL_ROWS) * -(-cols // PANEL_COLS)
        return panels * 8192, panels * 256
    code, scale = ctypes.c_int64(), ctypes.c_int64()
    _check(load_library().tabby_fp8_bytes(rows, cols, block_rows, ctypes.byref(code), ctypes.byref(scale)))
    return code.value, scale.value


class Fp8Matrix:
    """A [rows, cols] matrix in FP8 on the device, in the library's panel layout, a scale to each
    block of ``block_rows`` (1 or 128) x 128. Its buffers may be written again with
    ``quantize(x, out=matrix)``."""

    def __init__(self, rows: int, cols: int, block_rows: int = 1, device="cuda"):
        self.rows, self.cols, self.block_rows = int(rows), int(cols), int(block_rows)
        self._code_bytes, scale = sizes(self.rows, self.cols, self.block_rows)
        self.data = torch.empty(self._code_bytes + scale, dtype=torch.uint8, device=device)  # codes, then scales

    @property
    def codes(self):
        return self.data[:self._code_bytes]

    @property
    def scales(self):
        return self.data[self._code_bytes:].view(torch.float32)

    @classmethod
    def quantize(cls, x, block_rows: int = 1, out: Optional["Fp8Matrix"] = None, stream=None) -> "Fp8Matrix":
        """``x`` ([rows, cols] or [cols], float32, float16 or bfloat16) rounded to FP8: a block's scale
        is the smallest power of two (2^-126 at least) with max |x| <= 448 of it, values go to the nearest
        code (ties to even); a block with a NaN or an infinity becomes NaN. ``block_rows`` is 1 for
        activations, 128 for weights."""
        x = rows_of(x, "x")
        code = dtype_code(x.dtype)
        rows, cols = x.shape
        device = x.device
        if out is not None:
            if (out.rows, out.cols, out.block_rows) != (rows, cols, block_rows):
                raise ValueError(f"out is {out.rows} x {out.cols} in blocks of {out.block_rows} rows, x is {rows} x {cols}, "
                                 f"asked for blocks of {block_rows}")
            on_device(device, out.data)
        ctx, handle = call_on(device, stream)
        with ctx:
            m = cls(rows, cols, block_rows, device) if out is None else out
            at = m.data.data_ptr()
            _check(load_library().tabby_fp8_quantize_device(
                x.data_ptr(), code, rows, cols, x.stride(0), m.block_rows, at, at + m._code_bytes, handle))
        return m

    @classmethod
    def from_rowmajor(cls, codes, scales, stream=None) -> "Fp8Matrix":
        """A checkpoint's weights, repacked once: ``codes`` [rows, cols], uint8 or torch.float8_e4m3fn,
        ``scales`` float32 [ceil(rows / 128), ceil(cols / 128)], what a block's codes are multiplied by."""
        if not codes.is_cuda or not scales.is_cuda:
            raise ValueError("codes and scales must be device (cuda) tensors")
        if codes.dtype not in (torch.uint8, torch.float8_e4m3fn) or scales.dtype != torch.float32:
            raise ValueError(f"codes must be uint8 or float8_e4m3fn and scales float32, got {codes.dtype} and {scales.dtype}")
        if codes.dim() != 2 or codes.shape[0] < 1 or codes.shape[1] < 1:
            raise ValueError(f"codes must be [rows, cols], not empty, got {tuple(codes.shape)}")
        rows, cols = codes.shape
        blocks = (-(-rows // BLOCK), -(-cols // BLOCK))
        if tuple(scales.shape) != blocks:
            raise ValueError(f"scales must have shape {blocks}, got {tuple(scales.shape)}")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales must be contiguous")
        on_device(codes.device, scales)
        ctx, handle = call_on(codes.device, stream)
        with ctx:
            m = cls(rows, cols, BLOCK, codes.device)
            at = m.data.data_ptr()
            _check(load_library().tabby_fp8_pack_device(
                codes.data_ptr(), scales.data_ptr(), rows, cols, at, at + m._code_bytes, handle))
        return m

    def dequantize(self, dtype=None, out=None, stream=None):
        """The values that the codes stand for, [rows, cols]: code times scale in float32 (the default;
        exact where the scale is a power of two and the value no subnormal), rounded to ``dtype``."""
        rows, cols, device = self.rows, self.cols, self.data.device
        if out is None:
            dtype = dtype or torch.float32
            code = dtype_code(dtype)
        else:
            code = _result_code(out, dtype, rows, cols, device)
            out = rows_of(out, "out")
        ctx, handle = call_on(device, stream)
        with ctx:
            if out is None:
                out = torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)
            at = self.data.data_ptr()
            _check(load_library().tabby_fp8_dequantize_device(
                at, at + self._code_bytes, rows, cols, self.block_rows, out.data_ptr(), code, out.stride(0), handle))
        return out


def matmul(x, w: Fp8Matrix, bias=None, dtype=None, out=None, stream=None, fast_sums: bool = False):
    """x W^T (+ bias), [rows, w.rows] of ``dtype`` (float32 by default): ``w`` has square blocks, ``x``
    is an ``Fp8Matrix`` with blocks of one row or a float tensor ([rows, k] or [k]), which is quantised
    in the call and may share memory with ``out``. Products of codes are exact, their sums float32,
    rounded once to ``dtype``. ``fast_sums``, for float16 and bfloat16, lets more than 64 rows go through the
    matrix cores as codes, at twice the rate: eight products at a time are added to 2^-13 of the largest of
    them."""
    device = w.data.device
    if w.block_rows != BLOCK:
        raise ValueError(f"the weights must have blocks of {BLOCK} rows, got {w.block_rows}")
    quantized = isinstance(x, Fp8Matrix)
    if not quantized:
        x = rows_of(x, "x")
        x_code = dtype_code(x.dtype)
        on_device(device, x)
    else:
        if x.block_rows != 1:
            raise ValueError(f"x must have blocks of one row, got {x.block_rows}")
        on_device(device, x.data)
    rows, k = (x.rows, x.cols) if quantized else x.shape
    if k != w.cols:
        raise ValueError(f"x has {k} columns, the weights {w.cols}")
    n = w.rows
    bias_at = None
    if bias is not None:
        on_device(device, bias)
        if bias.dtype != torch.float32 or not bias.is_contiguous() or tuple(bias.shape) != (n,):
            raise ValueError(f"bias must be a contiguous float32 tensor of {n} entries")
        bias_at = bias.data_ptr()
    if out is None:
        dtype = dtype or torch.float32
        code = dtype_code(dtype)
    else:
        code = _result_code(out, dtype, rows, n, device)
        out = rows_of(out, "out")
    if fast_sums:
        code |= FAST_SUMS
    lib = load_library()
    w_at = w.data.data_ptr()
    ctx, handle = call_on(device, stream)
    with ctx:
        if out is None:
            out = torch.empty_strided((rows, n), (n, 1), dtype=dtype, device=device)
        if quantized:
            x_at = x.data.data_ptr()
            _check(lib.tabby_fp8_matmul_device(
                x_at, x_at + x._code_bytes, rows, w_at, w_at + w._code_bytes, bias_at, n, k, out.data_ptr(), code,
                out.stride(0), handle))
        else:
            size = sum(sizes(rows, k, 1))
            space = torch.empty(size, dtype=torch.uint8, device=device)
            _check(lib.tabby_fp8_linear_device(
                x.data_ptr(), x_code, x.stride(0), rows, w_at, w_at + w._code_bytes, bias_at, n, k, out.data_ptr(),
                code, out.stride(0), space.data_ptr(), size, handle))
    return out


class LmHeadFp8:
    """An lm_head with FP8 weights [vocab, hidden] in square blocks and an optional float32 bias [vocab]."""

    def __init__(self, weight: Fp8Matrix, bias=None):
        if weight.block_rows != BLOCK:
            raise ValueError(f"the weights must have blocks of {BLOCK} rows, got {weight.block_rows}")
        self.weight, self.bias = weight, bias
        self.vocab, self.hidden = weight.rows, weight.cols

    def logits(self, hidden_states, dtype=None, out=None, stream=None, fast_sums: bool = False):
        """Logits [rows, vocab] (float32 by default) of hidden states [rows, hidden] or [hidden]; ``fast_sums`` as
        in ``matmul``."""
        return matmul(hidden_states, self.weight, self.bias, dtype=dtype, out=out, stream=stream, fast_sums=fast_sums)
